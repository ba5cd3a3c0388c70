"""Divergence from a teacher's list and its gradient for every kind of list, against 64 bits.

Tolerances: the sums of weights are off by REL of themselves (the derivation stands in test_gpu_logits.py), so a
logarithm by REL, for the listed tokens and for the rest's class; the loss is rounded to 32 bits.  Sums over the list
are 64-bit ones."""

import math

import numpy as np
import pytest
import torch

from _divergence import divergence

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
REL = 1e-5


@pytest.fixture
def ops():
    from mlxturbo_b200 import ops

    return ops


def check(ops, x, tv, ti, T=1.0, lse=None, weight=None):
    """Loss and gradient of all calls against 64 bits."""
    rows = x.shape[0]
    w = torch.ones(rows, device="cuda") if weight is None else weight
    kw = dict(temperature=T, teacher_logsumexp=lse)
    leaf = x.detach().clone().requires_grad_()
    loss = ops.distill_loss(leaf, tv, ti, **kw)
    (grad,) = torch.autograd.grad(loss, leaf, w)
    loss = loss.detach()
    loss1, grad1 = ops.distill_loss_and_grad(x, tv, ti, weight, **kw)
    assert torch.equal(ops.distill_loss(x, tv, ti, **kw), loss)
    fin = torch.finfo(x.dtype)
    for r in range(rows):
        want, g, size = divergence(x[r], tv[r], ti[r], T, None if lse is None else float(lse[r]), float(w[r]))
        for got in (float(loss[r]), float(loss1[r])):
            assert got == want or abs(got - want) <= 2 * REL + 2 ** -23 * abs(want) < math.inf, (r, got, want)
        bound = fin.eps / 2 * np.abs(g) + 2.01 * REL * size + fin.smallest_normal * fin.eps / 2
        for d in (grad, grad1):
            err = np.abs(d[r].double().cpu().numpy() - g)
            assert (err <= bound).all(), (r, float((err / bound).max()))
    return loss1


def student(rows, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    teacher = torch.randn((rows, V), generator=g) * 3
    x = teacher + 0.5 * torch.randn((rows, V), generator=g)
    return x.to(dtype).cuda(), teacher.to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V,k", [(40, 12), (3001, 12), (3001, 130)])
def test_repeated_ids(ops, V, k, tail, dtype):
    """Ids listed twice and more, beside empty places, empty lists, values of -inf and any order of the list."""
    x, teacher = student(9, V, dtype, V + k)
    tv, ti, lse = ops.topk(teacher, min(k, V), logsumexp=True)
    ti[0, 3:] = -1
    ti[1] = -1
    ti[2, 5:] = ti[2, 4]
    ti[3] = ti[3, 0]
    tv[2:5] -= math.log(k) + 1  # as often as k times the same id: its mass stays below 1
    ti[4, 1::2] = ti[4, ::2]
    tv[5, 2:7] = -torch.inf
    tv[6] = -torch.inf
    ti[7], tv[7] = ti[7].flip(0), tv[7].flip(0)
    ti[8, 1], ti[8, 2], ti[8, 5] = V, 2 ** 40, ti[8, 0]
    tv[8] -= 1
    if tail:
        lse[6] = -torch.inf  # nothing of the teacher's row is left
    weight = torch.tensor([1.0, 1.0, 1.0, 0.5, -2.0, 1.0, 1.0, 0.0, 1.0]).cuda()
    loss = check(ops, x, tv, ti, 1.0, lse if tail else None, weight)
    check(ops, x, tv.float(), ti.clamp(-1, V).int(), 2.0, lse if tail else None)
    assert float(loss[6]) == 0.0 and (loss >= -2 * REL).all()  # a divergence


def test_an_id_in_equal_parts(ops):
    """However an id's probability is cut into entries, the divergence is the same: none here."""
    x = torch.full((3, 500), -40.0, device="cuda")
    x[:, 7] = 10.0
    ti = torch.tensor([[7, 7, 7, 7], [7, 7, -1, -1], [7, -1, -1, -1]]).cuda()
    tv = torch.zeros((3, 4), device="cuda")
    lse = torch.tensor([4.0, 2.0, 1.0]).log().cuda()
    for kw in (dict(), dict(teacher_logsumexp=lse)):
        loss, grad = ops.distill_loss_and_grad(x, tv, ti, **kw)
        assert loss.abs().max() <= 2 * REL and grad.abs().max() <= 2 * REL


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", [None, "lowest", "inf"])
@pytest.mark.parametrize("V,k,T", [(40, 40, 1.0), (9, 9, 2.5), (300, 30, 0.7)])
def test_lists_of_all_that_is_left(ops, V, k, T, mask, dtype):
    """Small vocabularies and constrained answers: a list of all tokens that have any probability.  What the given
    log-sum-exp's rounding leaves of 1 is no rest; a rest beyond that stays an infinite loss."""
    rows = 64
    x, teacher = student(rows, V, dtype, V)
    if mask is None:
        k = V
    else:
        allowed = torch.zeros((rows, V), dtype=torch.bool, device="cuda")
        allowed.scatter_(1, uniform_ids(rows, V, k).cuda(), True)
        low = torch.finfo(dtype).min if mask == "lowest" else -torch.inf
        x, teacher = x.masked_fill(~allowed, low), teacher.masked_fill(~allowed, low)
    tv, ti, lse = ops.topk(teacher, k, logsumexp=True, temperature=T)
    for given in (lse, torch.logsumexp(teacher.float() / T, -1)):
        loss = check(ops, x, tv, ti, T, given)
        assert loss.isfinite().all() and (loss >= -2 * REL).all()
    if mask != "lowest":
        loss, grad = ops.distill_loss_and_grad(x, tv, ti, temperature=T, teacher_logsumexp=lse + 0.1)
        assert (loss == torch.inf).all() and grad.isfinite().all()


def uniform_ids(rows, V, k):
    g = torch.Generator().manual_seed(rows + V)
    return torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(rows)])


@pytest.mark.parametrize("rows,first", [(1, 0), (1, 3), (0, 0)])
def test_last_chunk_in_place(ops, rows, first):
    """A chunk of one row of a wider buffer is contiguous whatever its row stride, and may hold its own gradient."""
    V = 700
    buf = torch.randn((4, V + 20), generator=torch.Generator().manual_seed(1)).cuda()
    x = buf[first:first + rows, :V]
    assert x.is_contiguous()
    keep = buf.clone()
    tv, ti = ops.topk(keep[first:first + rows, :V].contiguous() * 0.9, 6)
    loss, grad = ops.distill_loss_and_grad(keep[first:first + rows, :V], tv, ti)
    again, out = ops.distill_loss_and_grad(x, tv, ti, out=x)
    assert out is x and torch.equal(loss, again)
    keep[first:first + rows, :V] = grad
    assert torch.equal(buf, keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [3000, 70003])
def test_masks_of_any_size(ops, V, tail, dtype):
    """Stretches of a row that a mask fills with one huge number: against its own maximum a stretch's sum may be
    anything, beside the row's it is nothing."""
    sizes = [s for s in (1e4, 1e9, 1e10, 3e20, 1e30, 2.9e38, 3.3e38) if s <= torch.finfo(dtype).max]
    x, teacher = student(6, V, dtype, V)
    hide = torch.rand((6, V), generator=torch.Generator().manual_seed(2)) < 0.7
    hide[:, 50:V // 2] = True
    hide[1, 60:] = True
    hide = hide.cuda()
    for size in sizes:
        for T in (0.3, 1.0, 2.0, 4.0):
            low = -torch.tensor(size, dtype=dtype).item()
            y, t = x.masked_fill(hide, low), teacher.masked_fill(hide, low)
            tv, ti, lse = ops.topk(t, 8, logsumexp=True, temperature=T)
            check(ops, y, tv, ti, T, lse if tail else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [2, 500, 40001])
def test_lists_of_masked_tokens(ops, V, tail, dtype):
    """All listed tokens masked in the model's row: an infinite loss with a finite gradient, or a loss of what is left
    where the teacher gives them nothing either."""
    x, teacher = student(5, V, dtype, V)
    k = min(V - 1, 6)
    tv, ti, lse = ops.topk(teacher, k, logsumexp=True)
    x.scatter_(1, ti, -torch.inf)
    x[3].scatter_(0, ti[3, :1], 1.0)  # all but one
    ti[1, 1:], tv[1, :1] = -1, -torch.inf
    ti[2] = -1
    tv[4] = -torch.inf
    loss = check(ops, x, tv, ti, 1.0, lse if tail else None)
    assert float(loss[0]) == math.inf
    for r in (1, 2, 4):
        assert float(loss[r]) < 1e-4 or (tail and V == 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [3000, 70003])
def test_rows_of_huge_logits(ops, V, tail, dtype):
    """Rows masked throughout with a huge number, their list among them, and rows whose live logits are all that
    large: 64 bits of l / T itself would hold none of the differences."""
    x, teacher = student(4, V, dtype, V)
    k = 8
    for size in (1e4, 1e9, 1e10, 3e20, 1e30, 2.9e38, 3.3e38):
        if size > torch.finfo(dtype).max:
            continue
        low = -torch.tensor(size, dtype=dtype).item()
        for T in (0.3, 1.0, 2.0, 4.0):
            tv, ti, lse = ops.topk(teacher, k, logsumexp=True, temperature=T)
            lse += 0.5  # the tokens not listed have a share
            y = x.clone()
            y[0] = low
            y[1] = -low
            y[2, ::2] = low
            y[2, 1::2] = low * (1 + 2 ** -6)
            y[2].scatter_(0, ti[2], low)
            y[3] = -low
            y[3, V // 3:V // 2] = 0.0
            y[3].scatter_(0, ti[3], -low)
            check(ops, y, tv, ti, T, lse if tail else None)


@pytest.mark.parametrize("tail", [False, True])
def test_captured_loss_and_backward_pass(ops, tail):
    """Loss and gradient through autograd in one captured graph, replayed on other logits, lists and weights."""
    rows, V, k = 7, 5001, 9
    first, second = (student(rows, V, torch.bfloat16, s) for s in (1, 2))
    lists = [ops.topk(t, k, logsumexp=True) for _, t in (first, second)]
    weights = [torch.rand(rows, generator=torch.Generator().manual_seed(s)).cuda() for s in (3, 4)]

    def step(x, tv, ti, lse, w):
        loss = ops.distill_loss(x, tv, ti, teacher_logsumexp=lse if tail else None)
        return loss.detach(), torch.autograd.grad(loss, x, w)[0]

    leaf = first[0].clone().requires_grad_()
    tv, ti, lse, w = (t.clone() for t in (*lists[0], weights[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf, tv, ti, lse, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step(leaf, tv, ti, lse, w)
    for (x, _), (v, i, s), wt in zip((second, first), lists[::-1], weights[::-1]):
        leaf.detach().copy_(x)
        for a, b in zip((tv, ti, lse, w), (v, i, s, wt)):
            a.copy_(b)
        graph.replay()
        want = step(x.clone().requires_grad_(), v, i, s, wt)
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])
