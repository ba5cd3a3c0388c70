"""Refusals of the operators on rows of logits, without a GPU (the pointers stand for nothing): arrays that a call may
leave out, given and misaligned, which the kernels read in whole elements, and drafts too long to be looked through."""

import ctypes

import pytest

from mlxturbo_b200 import _lib

P, ODD = 1 << 20, (1 << 20) + 2


def sample(t=None, k=None, p=None, m=None):
    return _lib.load().qmm_sample(P, 100, 2, 100, 0, P, t, 1.0, k, 0, p, 1.0, m, 0.0, P, None)


def topk(lse=None):
    return _lib.load().qmm_topk(P, 100, 2, 100, 0, 5, 1.0, P, P, lse, None)


def speculative(t=None, td=None):
    lib = _lib.load()
    need = lib.qmm_speculative_sample_workspace_size(2, 3)
    return lib.qmm_speculative_sample(P, 400, 100, P, 300, 100, 2, 3, 100, 0, P, P, t, 1.0, td, 1.0, P, P, P,
                                      ctypes.c_size_t(need), None)


def loss(lse=None, stats=None):
    return _lib.load().qmm_distill_loss(P, 100, 2, 100, 0, P, 0, P, 8, lse, 5, 1.0, P, stats, None)


def both(lse=None, weight=None):
    return _lib.load().qmm_distill_loss_grad(P, 100, 2, 100, 0, P, 0, P, 8, lse, 5, 1.0, weight, P, 2 * P, 100, None)


def backward(lse=None):
    return _lib.load().qmm_distill_backward(P, 100, 2, 100, 0, P, 0, P, 8, lse, 5, 1.0, P, P, 2 * P, 100, None)


@pytest.mark.parametrize("call,name", [(sample, n) for n in "tkpm"] + [(topk, "lse"), (speculative, "t"), (speculative, "td"),
                                       (loss, "lse"), (loss, "stats"), (both, "lse"), (both, "weight"), (backward, "lse")])
def test_misaligned_arrays(call, name):
    assert call(**{name: ODD}) == _lib.QMM_EINVAL
    assert b"misaligned" in _lib.load().qmm_last_error()


def test_longest_draft():
    """Each row's warp looks through the ids before it: lengths whose square would take minutes are refused."""
    lib = _lib.load()
    rc = lib.qmm_speculative_sample(P, 1 << 20, 4, P, 1 << 20, 4, 1, (1 << 16) + 1, 4, 0, P, P, None, 1.0, None, 1.0, P, P,
                                    P, ctypes.c_size_t(1 << 40), None)
    assert rc == _lib.QMM_EUNSUPPORTED and b"drafted" in lib.qmm_last_error()
