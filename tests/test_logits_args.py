"""Refusals of the operators on rows of logits, without a GPU: bad arguments are reported before any device work
(the pointers stand for nothing)."""

import ctypes
import math

import pytest
import torch

from mlxturbo_b200 import _lib

P = 1 << 20
NAMES = ["sample", "topk", "speculative_sample", "distill_loss", "distill_backward", "distill_loss_grad",
         "distill_loss_grad_out"]


@pytest.mark.parametrize("name", NAMES)
def test_registered_per_device(name):
    assert _lib.torch_ops() is not None
    has = lambda key: torch._C._dispatch_has_kernel_for_dispatch_key(f"mlxturbo_b200::{name}", key)  # noqa: E731
    assert has("CUDA") and has("CPU") and not has("CompositeImplicitAutograd")


def refused(rc, status, text=b""):
    assert rc == status and text in _lib.load().qmm_last_error(), (rc, _lib.load().qmm_last_error())


def sample(logits=P, stride=100, rows=2, V=100, dtype=0, u=P, t=1.0, k=0, p=1.0, m=0.0, ids=P):
    return _lib.load().qmm_sample(logits, stride, rows, V, dtype, u, None, t, None, k, None, p, None, m, ids, None)


def test_sample_arguments():
    assert sample(rows=0) == _lib.QMM_OK
    for bad in (dict(V=0), dict(rows=-1), dict(stride=-1), dict(k=-1), dict(p=0.0), dict(p=1.5), dict(p=math.nan),
                dict(m=-0.1), dict(m=1.5), dict(m=math.nan), dict(t=-1.0), dict(t=math.nan), dict(t=math.inf),
                dict(t=1e-9), dict(logits=None), dict(logits=P + 1), dict(u=None), dict(u=P + 2), dict(ids=P + 4)):
        refused(sample(**bad), _lib.QMM_EINVAL, b"sample")
    for bad in (dict(dtype=3), dict(dtype=-1), dict(V=1 << 31), dict(V=(1 << 32) + 100), dict(rows=1 << 40)):
        refused(sample(**bad), _lib.QMM_EUNSUPPORTED, b"sample")


def topk(logits=P, stride=100, rows=2, V=100, dtype=0, k=5, t=1.0, values=P, ids=P):
    return _lib.load().qmm_topk(logits, stride, rows, V, dtype, k, t, values, ids, None, None)


def test_topk_arguments():
    assert topk(rows=0) == _lib.QMM_OK
    for bad in (dict(k=0), dict(k=101), dict(k=-1), dict(t=0.0), dict(t=math.nan), dict(V=-1), dict(logits=P + 1),
                dict(values=P + 1), dict(ids=None)):
        refused(topk(**bad), _lib.QMM_EINVAL, b"topk")
    for bad in (dict(V=5000, k=1025), dict(dtype=9), dict(V=1 << 31, k=4)):
        refused(topk(**bad), _lib.QMM_EUNSUPPORTED, b"topk")


def spec(logits=P, draft=P, B=2, n=3, V=100, dtype=0, ids=P, u=P, t=1.0, td=1.0, tokens=P, ws=P, size=None, stride=100):
    lib = _lib.load()
    need = lib.qmm_speculative_sample_workspace_size(B, n) if size is None else size
    return lib.qmm_speculative_sample(logits, 400, stride, draft, 300, 100, B, n, V, dtype, ids, u, None, t, None, td,
                                      tokens, P, ws, ctypes.c_size_t(need), None)


def test_speculative_arguments():
    lib = _lib.load()
    assert spec(B=0) == _lib.QMM_OK
    assert lib.qmm_speculative_sample_workspace_size(4, 3) >= 4 * 7 * 16
    assert lib.qmm_speculative_sample_workspace_size(-1, 3) == 0
    for bad in (dict(n=-1), dict(V=0), dict(t=-1.0), dict(td=math.nan), dict(draft=None), dict(ids=None), dict(u=P + 1),
                dict(tokens=P + 4), dict(ws=None), dict(ws=P + 8), dict(size=16), dict(stride=-4)):
        refused(spec(**bad), _lib.QMM_EINVAL, b"speculative_sample")
    for bad in (dict(dtype=4), dict(B=1 << 26, n=7), dict(n=1 << 40), dict(V=1 << 31)):
        refused(spec(**bad, size=1 << 40), _lib.QMM_EUNSUPPORTED, b"speculative_sample")


def distill(which="loss", logits=P, stride=100, rows=2, V=100, dtype=0, tv=P, tdt=0, ti=P, idb=8, k=5, t=1.0, loss=P,
            stats=P, grad=2 * P, gstride=100):
    lib = _lib.load()
    head = (logits, stride, rows, V, dtype, tv, tdt, ti, idb, None, k, t)
    if which == "loss":
        return lib.qmm_distill_loss(*head, loss, stats, None)
    if which == "both":
        return lib.qmm_distill_loss_grad(*head, None, loss, grad, gstride, None)
    return lib.qmm_distill_backward(*head, stats, loss, grad, gstride, None)


@pytest.mark.parametrize("which", ["loss", "both", "backward"])
def test_distill_arguments(which):
    assert distill(which, rows=0) == _lib.QMM_OK
    bad = [dict(k=0), dict(idb=2), dict(t=0.0), dict(t=math.inf), dict(V=0), dict(logits=P + 1), dict(tv=None),
           dict(tv=P + 2, tdt=2), dict(ti=P + 4), dict(loss=P + 1)]
    if which != "both":
        bad.append(dict(stats=P + 8))
    if which != "loss":
        bad += [dict(grad=None), dict(gstride=99)]
    if which == "both":
        bad.append(dict(grad=P, stride=200))  # over the logits, but not row for row
    if which == "backward":
        bad += [dict(grad=P), dict(stats=None)]
    for b in bad:
        refused(distill(which, **b), _lib.QMM_EINVAL, b"distill")
    for b in (dict(dtype=5), dict(tdt=7), dict(k=513), dict(V=1 << 31)):
        refused(distill(which, **b), _lib.QMM_EUNSUPPORTED, b"distill")


def test_rows_too_long_for_the_marks_of_a_list():
    """teacher_logsumexp needs a byte of shared memory to 16 bytes of a CTA's part of a row."""
    V = 1 << 24
    rc = _lib.load().qmm_distill_loss(P, V, 2, V, _lib.QMM_F32, P, 0, P, 8, P, 5, 1.0, P, None, None)
    refused(rc, _lib.QMM_EUNSUPPORTED, b"too long")


def test_all_cpu_arguments_are_refused():
    from mlxturbo_b200 import ops

    x, u = torch.randn(4, 64), torch.rand(4)
    ids = torch.zeros(4, 3, dtype=torch.int64)
    for call in (lambda: ops.sample(x, u), lambda: ops.topk(x, 3),
                 lambda: ops.speculative_sample(x[None], x[None, :3], ids[:1], u[None]),
                 lambda: ops.distill_loss(x, x[:, :3], ids), lambda: ops.distill_loss_and_grad(x, x[:, :3], ids)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_gradients_that_are_not_there_are_refused():
    from mlxturbo_b200 import ops

    x = torch.randn(4, 64)
    tv, ids = torch.randn(4, 3).requires_grad_(), torch.zeros(4, 3, dtype=torch.int64)
    with pytest.raises(NotImplementedError, match="teacher"):
        ops.distill_loss(x, tv, ids)
    with pytest.raises(NotImplementedError, match="autograd"):
        ops.distill_loss_and_grad(x.requires_grad_(), tv.detach(), ids)


@pytest.mark.gpu
def test_tensor_arguments():
    from mlxturbo_b200 import ops

    x, u = torch.randn(4, 64, device="cuda"), torch.rand(4, device="cuda")
    ids = torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    tv, ti = ops.topk(x, 3)
    draft = x[None, :3]
    bad = [lambda: ops.sample(x, u[:3]), lambda: ops.sample(x, u.double()), lambda: ops.sample(x, u.cpu()),
           lambda: ops.sample(x, u, top_p=u[:3]), lambda: ops.sample(x, u, top_k=u), lambda: ops.sample(x, u, top_p=0.0),
           lambda: ops.sample(x, u, temperature=torch.ones(4)), lambda: ops.sample(x[:, :0], u),
           lambda: ops.topk(x, 65), lambda: ops.topk(x, 0), lambda: ops.topk(x, -1),
           lambda: ops.speculative_sample(x[None], draft, ids[:1], u[None, :3]),
           lambda: ops.speculative_sample(x[None], draft.half(), ids[:1], u[None]),
           lambda: ops.speculative_sample(x[None], draft[..., :5], ids[:1], u[None]),
           lambda: ops.speculative_sample(x[None], draft, ids[:1].float(), u[None]),
           lambda: ops.distill_loss(x, tv[:3], ti[:3]), lambda: ops.distill_loss(x, tv, ti[:, :2]),
           lambda: ops.distill_loss(x, tv, ti.short()), lambda: ops.distill_loss(x, tv, ti, temperature=0.0),
           lambda: ops.distill_loss(x, tv, ti, teacher_logsumexp=u[:2]), lambda: ops.distill_loss(x, tv[:, :0], ti[:, :0]),
           lambda: ops.distill_loss_and_grad(x, tv, ti, u.double()),
           lambda: ops.distill_loss_and_grad(x, tv, ti, out=x.half()),
           lambda: ops.distill_loss_and_grad(x, tv, ti, out=x.t().contiguous().t()),
           lambda: ops.distill_loss_and_grad(x[1:3], tv[:2], ti[:2], out=x[2:4])]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for call in (lambda: ops.sample(x.double(), u), lambda: ops.sample(x.long(), u), lambda: ops.topk(x.double(), 3),
                 lambda: ops.topk(torch.randn(1, 3000, device="cuda"), 1025),
                 lambda: ops.distill_loss(x, torch.zeros(4, 600, device="cuda"),
                                          torch.zeros(4, 600, dtype=torch.int64, device="cuda"))):
        with pytest.raises(NotImplementedError):
            call()
