"""Sizes beyond what the kernels can index are refused before anything is launched (no GPU: the pointers stand
for nothing, and a call that went on would end with a CUDA error)."""

import ctypes

import pytest

from mlxturbo_b200 import _lib

P = 1 << 20  # 256-byte aligned


def mx_gather(rows, E, sorted_ids, N=8, K=32, x_rows=1024, lhs=P):
    lib = _lib.load()
    need = lib.qmm_mx_gather_workspace_size(rows, E, N, K, _lib.QMM_BF16, 0, sorted_ids)
    return lib.qmm_mx_gather(P, None, P, P, lhs, P, P, rows, x_rows, E, N, K, _lib.QMM_BF16, sorted_ids, P, need, None)


@pytest.mark.parametrize("rows,E", [(34_000_000, 16384), (600_000_000, 1000), (700_000_000, 16384)])
def test_unsorted_ids_past_the_sort(rows, E):
    """The sort counts (E + 1) x rows / 256 cells in 32 bits."""
    lib = _lib.load()
    assert (E + 1) * ((rows + 255) // 256) >= 2 ** 31
    assert mx_gather(rows, E, 0) == _lib.QMM_EUNSUPPORTED and b"beyond limits" in lib.qmm_last_error()
    need = lib.qmm_sort_workspace_size(rows, E)
    rc = lib.qmm_sort_rows(P, rows, E, 1, P, P, P, P, P, need, None)
    assert rc == _lib.QMM_EUNSUPPORTED and b"sort_rows" in lib.qmm_last_error()


def test_more_rows_than_an_int():
    lib = _lib.load()
    rows = (1 << 32) + 256  # 256 in 32 bits
    rc = lib.qmm_sort_rows(P, rows, 4, 1, P, P, P, P, P, ctypes.c_size_t(1 << 40), None)
    assert rc == _lib.QMM_EUNSUPPORTED


@pytest.mark.parametrize("rows,E", [(1 << 30, 4), (800_000_000, 8)])
def test_rows_past_the_planes(rows, E):
    assert mx_gather(rows, E, 1) == _lib.QMM_EUNSUPPORTED
