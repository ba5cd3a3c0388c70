"""Rows of logits: sampling, top-k, speculative acceptance and distillation against plain forms in 64 bits.

Token ids and counts are compared exactly.  Log-sum-exps, losses and gradients are in 32 bits: a weight
2^(x - m) log2(e) / T is off by a rounding of its difference, of its exponent (|a| ln 2 2^-23, |a| < 60 here) and of
ex2 (2^-22), a sum by less than 2^-16 of itself (the kernels' own bound; 1e-5 is taken for the sums of these sizes:
at most 40 roundings of 2^-24, the mean exponent below 20, 8 rescalings of 2^-22)."""

import numpy as np
import pytest
import torch

import _logits as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
REL = 1e-5  # of a sum or a weight, see above


@pytest.fixture
def ops():
    from mlxturbo_b200 import ops

    return ops


def make(rows, V, dtype, seed, spread=2.0, peaks=8):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, V), generator=g) * spread
    n = min(peaks, V)
    at = torch.stack([torch.randperm(V, generator=g)[:n] for _ in range(rows)])
    x.scatter_(1, at, 8 + 3 * torch.randn((rows, n), generator=g))
    return x.to(dtype).cuda()


def uniform(seed, *shape):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed)).cuda()


SETTINGS = [dict(), dict(temperature=0.7, top_k=5), dict(temperature=1.3, top_p=0.8),
            dict(temperature=0.9, min_p=0.05), dict(temperature=0.8, top_k=50, top_p=0.9, min_p=0.02),
            dict(top_p=0.95, min_p=0.001), dict(temperature=2.5, top_k=700, top_p=0.99), dict(temperature=0.0),
            dict(temperature=1.0, top_k=1), dict(top_p=1e-6), dict(min_p=1.0)]


def as_row(s):
    return {"T": s.get("temperature", 1.0), **{k: v for k, v in s.items() if k != "temperature"}}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 33, 1000, 4097, 32001])
def test_sample_settings(ops, V, dtype):
    x, u = make(6, V, dtype, V), uniform(V + 1, 6)
    for s in SETTINGS:
        got = ops.sample(x, u, **s)
        assert got.dtype == torch.int64 and got.shape == (6,)
        assert got.tolist() == [R.sample(x[r], u[r], **as_row(s)) for r in range(6)], s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 20])
def test_sample_large_vocabulary(ops, rows, dtype):
    V = 248320
    x, u = make(rows, V, dtype, rows), uniform(rows, rows)
    for s in SETTINGS[:7] + [dict(temperature=3.0, top_p=0.9), dict(temperature=2.0, top_k=100000),
                             dict(temperature=2.0, top_k=5000, top_p=0.7, min_p=0.001)]:
        got = ops.sample(x, u, **s)
        assert got.tolist() == [R.sample(x[r], u[r], **as_row(s)) for r in range(rows)], s


@pytest.mark.parametrize("spread", [0.0, 0.01, 1.0])
def test_sample_flat_rows(ops, spread):
    """No token stands out: borders lie among thousands of equal or nearly equal weights."""
    V = 20011
    x = (torch.randn((4, V), generator=torch.Generator().manual_seed(3)) * spread).bfloat16().cuda()
    u = torch.tensor([0.0, 0.25, 0.5, 1 - 2 ** -24]).cuda()
    for s in [dict(), dict(top_k=4096), dict(top_k=19999, top_p=0.5), dict(top_p=0.75), dict(min_p=0.5),
              dict(top_p=0.999, min_p=0.9), dict(top_k=3)]:
        got = ops.sample(x, u, **s)
        assert got.tolist() == [R.sample(x[r], u[r], **as_row(s)) for r in range(4)], s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 3001, 70000])
def test_sample_masks(ops, V, dtype):
    """-inf, the type's lowest value and NaN in masked places, rows that a mask leaves nothing or one token,
    infinite logits."""
    x = make(9, V, dtype, 7)
    g = torch.Generator().manual_seed(11)
    hide = (torch.rand((9, V), generator=g) < 0.7).cuda()
    x[0][hide[0]] = -torch.inf
    x[1][hide[1]] = torch.finfo(dtype).min
    x[2][hide[2]] = torch.nan
    x[3] = -torch.inf
    x[4] = -torch.inf
    x[4, V - 1] = -3.0
    x[5] = torch.nan
    x[6, V // 2] = torch.inf
    x[7, 0] = x[7, V - 2] = torch.inf
    x[8] = torch.finfo(dtype).min
    u = uniform(5, 9)
    for s in SETTINGS:
        got = ops.sample(x, u, **s)
        assert got.tolist() == [R.sample(x[r], u[r], **as_row(s)) for r in range(9)], s


def test_sample_per_row_settings(ops):
    rows, V = 40, 5000
    x, u = make(rows, V, torch.float16, 1), uniform(2, rows)
    g = torch.Generator().manual_seed(4)
    T = torch.rand(rows, generator=g) * 1.5
    T[::7] = 0
    T[3] = -1
    k = torch.randint(0, 60, (rows,), generator=g)
    k[5], k[6] = -3, 2 ** 40
    p = torch.rand(rows, generator=g) * 1.2
    p[9] = -0.5
    m = torch.rand(rows, generator=g) * 0.2 - 0.05
    got = ops.sample(x, u, temperature=T.cuda(), top_k=k.cuda(), top_p=p.cuda(), min_p=m.cuda())
    want = [R.sample(x[r], u[r], float(T[r]), int(k[r]), float(p[r]) if p[r] > 0 else 1e-30, float(m[r]))
            for r in range(rows)]
    assert got.tolist() == want
    # some numbers, some tensors, broadcast over the leading axes
    y = x.view(4, 10, V)
    got = ops.sample(y, u.view(4, 10), temperature=0.8, top_k=k[:10].cuda(), top_p=p[:4].clamp(0.1, 1).cuda()[:, None])
    want = [R.sample(x[r], u[r], 0.8, int(k[r % 10]), float(p[r // 10].clamp(0.1, 1))) for r in range(rows)]
    assert got.reshape(-1).tolist() == want


def test_sample_strides_and_alignment(ops):
    V = 1003
    base = make(12, 2 * V + 5, torch.bfloat16, 8)
    u = uniform(9, 12)
    for x in (base[:, 3:3 + V], base[:, 1::2][:, :V], base[2:3].expand(12, -1), base.t().contiguous().t()[:, :V]):
        for s in SETTINGS[:5]:
            assert ops.sample(x, u, **s).tolist() == [R.sample(x[r], u[r], **as_row(s)) for r in range(12)]
    assert ops.sample(base[0], u[0]).shape == ()
    assert ops.sample(base[:0], u[:0]).shape == (0,)


def test_sample_frequencies(ops):
    """Over many draws a token comes as often as it weighs (fixed numbers: 4096 evenly spaced u)."""
    x = torch.tensor([[1.0, 2.0, 0.5, -torch.inf, 1.5]]).cuda()
    n = 4096
    got = ops.sample(x.expand(n, -1), (torch.arange(n, device="cuda") + 0.5) / n)
    p = torch.softmax(x[0].double(), -1)
    count = torch.bincount(got, minlength=5).double() / n
    assert (count - p).abs().max() <= 1 / n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(1, 1), (5, 5), (8, 3), (1000, 1), (1000, 1000), (4097, 64), (32001, 20), (32001, 300),
                                 (50000, 1024), (248320, 20), (248320, 256), (248320, 1024)])
def test_topk(ops, V, k, dtype):
    x = make(3, V, dtype, V + k)
    values, ids, lse = ops.topk(x, k, logsumexp=True, temperature=0.7)
    assert values.dtype == dtype and ids.dtype == torch.int64 and lse.dtype == torch.float32
    for r in range(3):
        v, i = R.topk(x[r], k)
        assert ids[r].tolist() == i.tolist()
        assert values[r].double().tolist() == v.tolist()
        want = R.logsumexp(x[r], 0.7)
        assert abs(float(lse[r]) - want) <= REL + 2 ** -24 * abs(want)
    two = ops.topk(x, k)
    assert len(two) == 2 and torch.equal(two[1], ids)


@pytest.mark.parametrize("V,k", [(3000, 17), (3000, 1000), (100000, 50)])
def test_topk_ties_and_masks(ops, V, k):
    x = torch.zeros((7, V), dtype=torch.bfloat16)
    x[0, V // 2] = 1.0
    x[1] = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(1)).bfloat16()
    x[2] = -torch.inf
    x[3] = -torch.inf
    x[3, 7:7 + k // 2] = -2.0
    x[4, ::2] = torch.nan
    x[5, ::3] = -0.0
    x[6] = torch.inf
    x = x.cuda()
    values, ids, lse = ops.topk(x, k, logsumexp=True)
    for r in range(7):
        v, i = R.topk(x[r], k)
        assert ids[r].tolist() == i.tolist(), r
        assert values[r].double().tolist() == v.tolist(), r
        want = R.logsumexp(x[r])
        assert float(lse[r]) == want if np.isinf(want) else abs(float(lse[r]) - want) <= REL + 2 ** -24 * abs(want)


def test_topk_leading_axes_and_views(ops):
    base = make(12, 777, torch.float16, 2)
    x = base[:, 5:705].reshape(3, 4, 700)
    values, ids = ops.topk(x, 9)
    assert values.shape == ids.shape == (3, 4, 9)
    v, i = ops.topk(base[:, 5:705], 9)
    assert torch.equal(ids.view(12, 9), i) and torch.equal(values.view(12, 9), v)
    assert torch.equal(torch.gather(x, -1, ids), values)
    assert ops.topk(base[:0], 3)[1].shape == (0, 3)
    one = ops.topk(base[3], 4)
    assert torch.equal(one[1], ops.topk(base[3:4], 4)[1][0])


def spec_case(B, n, V, dtype, seed, closeness=0.9):
    logits = make(B * (n + 1), V, dtype, seed).view(B, n + 1, V)
    noise = torch.randn((B, n, V), generator=torch.Generator().manual_seed(seed + 1)).cuda()
    draft = (closeness * logits[:, :n].float() + 0.7 * noise).to(dtype)
    ids = torch.empty((B, n), dtype=torch.int64)
    u = torch.rand((B, n), generator=torch.Generator().manual_seed(seed + 2))
    for b in range(B):
        for i in range(n):
            ids[b, i] = R.sample(draft[b, i], u[b, i])
    return logits, draft, ids.cuda(), uniform(seed + 3, B, n + 1)


def check_spec(ops, logits, draft, ids, u, T=1.0, Td=None):
    tokens, accepted = ops.speculative_sample(logits, draft, ids, u, temperature=T, draft_temperature=Td)
    assert tokens.dtype == accepted.dtype == torch.int64
    for b in range(logits.shape[0]):
        t = float(T[b]) if torch.is_tensor(T) else T
        td = t if Td is None else float(Td[b]) if torch.is_tensor(Td) else Td
        want, j = R.speculative(logits[b], draft[b], ids[b], u[b], t, td)
        assert tokens[b].tolist() == want and int(accepted[b]) == j, b
    return accepted


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,n,V", [(1, 1, 5), (7, 3, 1000), (3, 8, 4097), (16, 4, 32001), (2, 40, 300)])
def test_speculative(ops, B, n, V, dtype):
    logits, draft, ids, u = spec_case(B, n, V, dtype, B + n + V)
    check_spec(ops, logits, draft, ids, u)
    check_spec(ops, logits, draft, ids, u, T=0.6, Td=0.9)
    check_spec(ops, logits, draft, ids, u, T=0.0)
    check_spec(ops, logits, draft, ids, u, T=0.0, Td=1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_speculative_large_vocabulary(ops, dtype):
    logits, draft, ids, u = spec_case(3, 4, 248320, dtype, 5)
    check_spec(ops, logits, draft, ids, u)
    logits, draft, ids, u = spec_case(1, 2, 248320, dtype, 6, closeness=0.3)
    check_spec(ops, logits, draft, ids, u, T=2.0)  # flat: borders closer than the fast sums' bound


def test_speculative_ends_masks_and_settings(ops):
    B, n, V = 12, 4, 3000
    logits, draft, ids, u = spec_case(B, n, V, torch.bfloat16, 21)
    ids[0, 0] = -1  # no draft at all
    ids[1, 2] = -7
    ids[2, 1], ids[2, 3] = V, 5
    logits[3, 0, int(ids[3, 0])] = -torch.inf  # the model never says it
    draft[4, 0] = -torch.inf  # a draft that gives nothing any probability
    logits[5, 0] = -torch.inf  # nothing to draw from
    logits[6, 1, ::2] = torch.finfo(torch.bfloat16).min
    draft[7, 0, ::3] = torch.nan
    logits[8] = draft[8, :1]  # the same distribution
    u[8, :n] = 1 - 2 ** -24
    u[9] = 0.0
    u[10] = 1 - 2 ** -24
    T = torch.linspace(0.4, 1.6, B).cuda()
    T[11] = 0
    check_spec(ops, logits, draft, ids, u)
    check_spec(ops, logits, draft, ids, u, T=T)
    check_spec(ops, logits, draft, ids, u, T=T, Td=T.flip(0))
    # rows of a wider buffer, and starts of other alignment on the two sides
    wide = torch.zeros((B, n + 1, 2 * V), dtype=torch.bfloat16, device="cuda")
    wide[..., 3:3 + V] = logits
    odd = torch.zeros((B, n, V + 1), dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = draft
    check_spec(ops, wide[..., 3:3 + V], odd[..., 1:], ids.int(), u)
    # no drafted position: a sample
    tokens, accepted = ops.speculative_sample(logits[:, :1], draft[:, :0], ids[:, :0], u[:, :1])
    assert torch.equal(tokens[:, 0], ops.sample(logits[:, 0], u[:, 0])) and not accepted.any()
    tokens, accepted = ops.speculative_sample(logits[0], draft[0], ids[0], u[0])
    assert tokens.shape == (n + 1,) and accepted.shape == ()


def distill_case(rows, V, k, dtype, seed, lse):
    teacher = make(rows, V, dtype, seed)
    x = (teacher.float() + 0.5 * torch.randn((rows, V), generator=torch.Generator().manual_seed(seed)).cuda()).to(dtype)
    return x, teacher, k, lse


def check_distill(ops, x, tv, ti, T=1.0, lse=None, weight=None, same_bits=True):
    """Loss and gradient of all three calls against 64 bits; same_bits: x starts where a copy of it does (the order
    of a sum's terms goes by 16-byte boundaries, so its last bits by where a row starts)."""
    rows, V = x.shape
    w = torch.ones(rows, device="cuda") if weight is None else weight
    kw = dict(temperature=T, teacher_logsumexp=lse)
    leaf = x.detach().clone().requires_grad_()
    loss = ops.distill_loss(leaf, tv, ti, **kw)
    (grad,) = torch.autograd.grad(loss, leaf, w)
    loss = loss.detach()
    loss1, grad1 = ops.distill_loss_and_grad(x, tv, ti, weight, **kw)
    inplace = x.clone()
    loss2, grad2 = ops.distill_loss_and_grad(inplace, tv, ti, weight, out=inplace, **kw)
    assert grad2 is inplace and grad.dtype == grad1.dtype == x.dtype
    plain = ops.distill_loss(x, tv, ti, **kw)
    assert not plain.requires_grad and torch.equal(plain, loss1) and torch.equal(loss, loss2)
    if same_bits:
        assert torch.equal(loss1.view(torch.int32), loss2.view(torch.int32)) and torch.equal(grad1, grad2)
    fin = torch.finfo(x.dtype)
    for r in range(rows):
        want, g, size = R.distill(x[r], tv[r], ti[r], T, None if lse is None else float(lse[r]), float(w[r]))
        for got in (loss, loss1):
            assert abs(float(got[r]) - want) <= 2 * REL + 2 ** -23 * abs(want) or float(got[r]) == want, (r, want)
        # a sum and a weight off by REL each, then one rounding to the type (or to its subnormals' grid)
        bound = fin.eps / 2 * np.abs(g) + 2.01 * REL * size + fin.smallest_normal * fin.eps / 2
        for got in (grad, grad1, grad2):
            err = np.abs(got[r].double().cpu().numpy() - g)
            assert (err <= bound).all(), (r, float((err / bound).max()))
    return loss


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V,k", [(2, 1), (9, 9), (1000, 20), (4097, 128), (32001, 64), (32001, 512)])
def test_distill(ops, V, k, tail, dtype):
    x, teacher, *_ = distill_case(4, V, k, dtype, V + k, tail)
    for T in (1.0, 2.5):
        tv, ti, lse = ops.topk(teacher, k, logsumexp=True, temperature=T)
        weight = torch.tensor([1.0, 0.0, 0.25, -2.0]).cuda()
        check_distill(ops, x, tv, ti, T, lse if tail else None, weight)
    check_distill(ops, x, tv.float(), ti.int(), 1.0, None, None)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_large_vocabulary(ops, tail):
    x, teacher, *_ = distill_case(2, 248320, 64, torch.bfloat16, 3, tail)
    tv, ti, lse = ops.topk(teacher, 64, logsumexp=True)
    check_distill(ops, x, tv, ti, 1.0, lse if tail else None)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_lists(ops, tail):
    """Empty places, an empty list, ids listed twice and more, values of -inf, in any order."""
    rows, V, k = 8, 3001, 12
    x, teacher, *_ = distill_case(rows, V, k, torch.float32, 17, tail)
    tv, ti, lse = ops.topk(teacher, k, logsumexp=True)
    ti[0, 3:] = -1
    ti[1] = -1
    ti[2, 5:] = ti[2, 4]
    ti[3] = ti[3, 0]
    tv[3] -= 3.0  # twelve times the same id: its mass stays below 1
    tv[4, 2:7] = -torch.inf
    tv[5] = -torch.inf
    ti[6] = ti[6].flip(0)
    tv[6] = tv[6].flip(0)
    ti[7, 1], ti[7, 2] = V, 2 ** 40
    lse = lse.clone()
    if tail:
        lse[5] = -torch.inf  # nothing of the teacher's row is left
    loss = check_distill(ops, x, tv, ti, 1.0, lse if tail else None)
    assert float(loss[5]) == 0.0
    if not tail:
        assert float(loss[1]) == 0.0


def test_distill_masked_student(ops):
    """Masked logits have no probability: -inf and the type's lowest value give the same, a listed one an
    infinite loss with a finite gradient, and a row of no weight zeros whatever it holds."""
    rows, V, k = 6, 2000, 8
    x, teacher, *_ = distill_case(rows, V, k, torch.bfloat16, 23, False)
    tv, ti = ops.topk(teacher, k)
    hide = torch.ones((rows, V), dtype=torch.bool, device="cuda").scatter_(1, ti, False)
    hide &= (torch.rand((rows, V), generator=torch.Generator().manual_seed(1)) < 0.8).cuda()
    y = x.masked_fill(hide, -torch.inf)
    low = x.masked_fill(hide, torch.finfo(torch.bfloat16).min)
    check_distill(ops, y, tv, ti)
    assert torch.equal(ops.distill_loss_and_grad(y, tv, ti)[1], ops.distill_loss_and_grad(low, tv, ti)[1])
    z = x.clone()
    z[0, ti[0, 2]] = -torch.inf
    z[1] = -torch.inf
    z[2, 5] = torch.nan
    z[3, 9] = torch.inf
    loss, grad = ops.distill_loss_and_grad(z, tv, ti)
    assert float(loss[0]) == torch.inf and grad[0].isfinite().all()
    assert loss[1:4].isnan().all() and grad[1:4].isnan().all() and loss[4:].isfinite().all()
    w = torch.zeros(rows, device="cuda")
    loss, grad = ops.distill_loss_and_grad(z, tv, ti, w)
    assert not grad.any() and float(loss[0]) == torch.inf
    leaf = z.clone().requires_grad_()
    (grad,) = torch.autograd.grad(ops.distill_loss(leaf, tv, ti), leaf, w)
    assert not grad.any()


def test_distill_far_apart(ops):
    """The tokens not listed hold a millionth of a billionth of the model's mass: their sum keeps its digits."""
    V, k = 4000, 4
    x = torch.randn((2, V), generator=torch.Generator().manual_seed(2)).cuda()
    ti = torch.tensor([[1, 5, 9, 13], [3999, 0, 2, 4]]).cuda()
    x.scatter_(1, ti, 45.0)
    tv = torch.tensor([[3.0, 2.0, 1.0, 0.0]] * 2).cuda()
    check_distill(ops, x, tv, ti, 1.0, torch.logsumexp(tv, -1) + 0.1)
    y = x.masked_fill(torch.ones_like(x, dtype=torch.bool).scatter_(1, ti, False), -torch.inf)
    loss, grad = ops.distill_loss_and_grad(y, tv, ti, teacher_logsumexp=torch.logsumexp(tv, -1) + 0.1)
    assert (loss == torch.inf).all() and grad.isfinite().all()


def test_distill_differences(ops):
    """The gradient against central differences of the loss, both in 32 bits."""
    rows, V, k = 2, 50, 6
    x, teacher, *_ = distill_case(rows, V, k, torch.float32, 31, False)
    tv, ti, lse = ops.topk(teacher, k, logsumexp=True)
    for kw in (dict(), dict(teacher_logsumexp=lse)):
        _, grad = ops.distill_loss_and_grad(x, tv, ti, **kw)
        h = 2.0 ** -5
        eye = torch.eye(V, device="cuda") * h
        for r in range(rows):
            args = (tv[r].expand(V, k), ti[r].expand(V, k))
            more = {n: t[r].expand(V) for n, t in kw.items()}
            up, down = ops.distill_loss(x[r] + eye, *args, **more), ops.distill_loss(x[r] - eye, *args, **more)
            # third derivatives of a log-sum-exp are below 1 in size: h^2 / 6 each, and for the rest class' second
            # log-sum-exp; two losses off by 2 REL + 2^-23 |loss| each
            scale = float(ops.distill_loss(x[r:r + 1], tv[r:r + 1], ti[r:r + 1]).abs()) + 1
            bound = 2 * h * h / 6 + (2 * REL + 2 ** -23 * scale) / h
            assert ((up - down) / (2 * h) - grad[r]).abs().max() <= bound


def test_a_step_of_all_of_them(ops):
    """An lm_head's logits: a draft is verified, the next token sampled, the draft distilled from the lists."""
    g = torch.Generator().manual_seed(40)
    K, V, n = 256, 4096, 3
    w, s, b = ops.quantize(torch.randn((V, K), generator=g).cuda() * 0.2, dtype=torch.bfloat16)
    x = torch.randn((n + 1, K), generator=g).bfloat16().cuda()
    logits = ops.quantized_matmul(x, w, s, b)
    draft = (logits[:n].float() + torch.randn((n, V), generator=g).cuda()).bfloat16()
    u = uniform(41, n)
    ids = ops.sample(draft, u, temperature=0.8)
    assert ids.tolist() == [R.sample(draft[i], u[i], 0.8) for i in range(n)]
    ua = uniform(42, n + 1)
    tokens, accepted = ops.speculative_sample(logits, draft, ids, ua, temperature=0.8)
    want, j = R.speculative(logits, draft, ids, ua, 0.8)
    assert tokens.tolist() == want and int(accepted) == j
    tv, ti, lse = ops.topk(logits[:n], 16, logsumexp=True)
    check_distill(ops, draft, tv, ti, 1.0, lse)
    _, keys = ops.quantized_matmul_argmax(x, w, s, b)
    assert torch.equal(ops.argmax_from_keys(keys), ops.sample(logits, ua, temperature=0))
    assert torch.equal(ops.topk(logits, 1)[1][:, 0], ops.argmax_from_keys(keys))


def test_captured_streams_and_repeats(ops):
    """Graph replays on new contents, two streams at once, and the same bits in every call."""
    rows, V, k = 12, 30011, 16
    x, teacher, *_ = distill_case(rows, V, k, torch.bfloat16, 50, True)
    u = uniform(51, rows)
    logits, draft, ids, us = spec_case(3, 3, V, torch.bfloat16, 52)

    def step(x, u, logits, draft):
        tv, ti, lse = ops.topk(x, k, logsumexp=True)
        loss, grad = ops.distill_loss_and_grad(x, tv, ti, u, teacher_logsumexp=lse)
        return [ops.sample(x, u, top_p=0.9), ops.sample(x, u), tv, ti, lse, loss, grad,
                *ops.speculative_sample(logits, draft, ids, us)]

    want = step(x, u, logits, draft)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(x, u, logits, draft), want))
    static = [t.clone() for t in (teacher, u.flip(0), logits.flip(0), draft.flip(0))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    with torch.cuda.graph(second):
        got2 = step(*static)
    for a, b in zip(static, (x, u, logits, draft)):
        a.copy_(b)
    graph.replay()
    second.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(got2, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                out.append(step(x, u, logits, draft))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in out for a, b in zip(o, want))


def test_rows_behind_the_last_are_left(ops):
    """What lies around inputs and outputs stays as it was; a row does not depend on its neighbours."""
    V = 501
    buf = torch.full((5, V + 9), 7.0, dtype=torch.bfloat16, device="cuda")
    x = buf[1:4, 3:3 + V]
    x.copy_(make(3, V, torch.bfloat16, 60))
    keep = buf.clone()
    tv, ti = ops.topk(x, 5)
    ops.sample(x, uniform(1, 3), top_p=0.7)
    loss, grad = ops.distill_loss_and_grad(x, tv, ti)
    assert torch.equal(buf, keep)
    flat = torch.full((4 * V,), 3.0, dtype=torch.bfloat16, device="cuda")
    out = flat[V:V + 2 * V].view(2, V)  # starts at an odd element
    ops.distill_loss_and_grad(x[:2].contiguous(), tv[:2], ti[:2], out=out)
    assert torch.equal(out, grad[:2]) and (flat[:V] == 3).all() and (flat[3 * V:] == 3).all()


def test_rows_far_apart(ops):
    """Rows more than 2^31 elements from each other."""
    V, k = 5000, 12
    buf = torch.zeros(2 ** 31 + 4096 + V, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((2, V), (2 ** 31 + 4091, 1), 5)
    x.copy_(make(2, V, torch.bfloat16, 70))
    u = uniform(71, 2)
    for s in SETTINGS[:5]:
        assert ops.sample(x, u, **s).tolist() == [R.sample(x[r], u[r], **as_row(s)) for r in range(2)]
    tv, ti, lse = ops.topk(x, k, logsumexp=True)
    close = x.contiguous()
    assert all(torch.equal(a, b) for a, b in zip((tv, ti, lse), ops.topk(close, k, logsumexp=True)))
    other = (x.float() + 0.1).bfloat16()
    for a, b in zip(ops.distill_loss_and_grad(x, tv, ti + 1, teacher_logsumexp=lse),
                    ops.distill_loss_and_grad(close, tv, ti + 1, teacher_logsumexp=lse)):
        assert torch.equal(a, b)
    got = ops.speculative_sample(x[:, None], other[:, None][:, :0], ti[:, :0], u[:, None])
    assert torch.equal(got[0][:, 0], ops.sample(x, u))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start", [1, 2, 3, 7])
def test_starts_of_every_alignment(ops, start, dtype):
    """Rows of an odd length that start at any element: each row's first and last vectors hold its neighbours'."""
    V, k = 1001, 9
    flat = make(1, 6 * V + start, dtype, 80 + start)[0]
    x = flat[start:start + 6 * V].view(6, V)
    u = uniform(3, 6)
    for s in SETTINGS[:6]:
        assert ops.sample(x, u, **s).tolist() == [R.sample(x[r], u[r], **as_row(s)) for r in range(6)]
    tv, ti, lse = ops.topk(x, k, logsumexp=True)
    for r in range(6):
        assert ti[r].tolist() == R.topk(x[r], k)[1].tolist()
    moved = ti.roll(1, 0)
    check_distill(ops, x, tv, moved, 1.0, lse, same_bits=False)
    check_distill(ops, x, tv, moved, 1.0, None, same_bits=False)
    ids = torch.stack([ti[0:2, 0], ti[1:3, 0]], 1)
    check_spec(ops, x.view(2, 3, V), make(4, V, dtype, 5).view(2, 2, V), ids, uniform(4, 2, 3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [24, 150])
def test_open_rows_of_a_batch(ops, rows, dtype):
    """Nucleus and plain sampling where thousands of tokens share the mass, in a batch of many rows, against 64-bit
    torch operations on the device; equal weights across the border among them."""
    V = 60000 if dtype == torch.float32 else 131072
    x = make(rows, V, dtype, 90, spread=1.8)
    x[::3] -= 0.0
    x[1::4] = (x[1::4] * 2).round() / 2  # few distinct values: hundreds of equal tokens
    u = uniform(91, rows)
    for T, p, k in ((1.0, 0.95, 0), (1.7, 0.8, 0), (0.8, 0.999, 0), (1.0, 1.0, 0), (1.0, 0.9, 300), (2.0, 0.97, 2000),
                    (1.3, 1.0, 5000), (2.0, 0.5, V // 3)):
        got = ops.sample(x, u, temperature=T, top_p=p, top_k=k)
        if k:  # a number a row goes to the same tokens
            ks = torch.full((rows,), k, device="cuda")
            assert torch.equal(got, ops.sample(x, u, temperature=T, top_p=p, top_k=ks))
        l = x.double()
        w = torch.exp((l - l.amax(-1, keepdim=True)) / T)
        if p < 1 or k:
            order = l.sort(dim=-1, descending=True, stable=True).indices
            ws = w.gather(-1, order)
            if k:
                ws[:, k:] = 0.0
            cum = ws.cumsum(-1)
            keep = torch.zeros_like(w, dtype=torch.bool).scatter_(-1, order, (ws > 0) & (cum - ws < p * cum[:, -1:]))
            w = torch.where(keep, w, 0.0)
        cum = w.cumsum(-1)
        want = (cum > u.double()[:, None] * cum[:, -1:]).to(torch.int8).argmax(-1)
        assert torch.equal(got, want), (T, p, k)


def test_second_derivative_is_refused(ops):
    x, teacher, *_ = distill_case(2, 500, 4, torch.float32, 5, False)
    tv, ti = ops.topk(teacher, 4)
    leaf = x.clone().requires_grad_()
    w = torch.ones(2, device="cuda", requires_grad=True)
    with pytest.raises(Exception, match="second derivative"):
        torch.autograd.grad(ops.distill_loss(leaf, tv, ti), leaf, w, create_graph=True)
    with torch.no_grad():
        assert not ops.distill_loss(leaf, tv, ti).requires_grad
    with torch.inference_mode():
        assert torch.equal(ops.distill_loss(x, tv, ti), ops.distill_loss(leaf, tv, ti).detach())
    loss = ops.distill_loss(leaf * 1.0, tv, ti)
    (loss * torch.tensor([2.0, 0.5], device="cuda")).sum().backward()
    again = x.clone().requires_grad_()
    want = torch.autograd.grad(ops.distill_loss(again, tv, ti), again, torch.tensor([2.0, 0.5], device="cuda"))[0]
    assert torch.equal(leaf.grad, want)


def test_tiny_and_huge_settings(ops):
    """Temperatures and filters at the ends of what is taken."""
    x, u = make(4, 3000, torch.float32, 6), uniform(7, 4)
    T = torch.tensor([1e-30, 1e-4, 1e6, 3e38]).cuda()
    m = torch.tensor([0.5, 1e-37, 0.999, 0.1]).cuda()
    for s in (dict(), dict(min_p=m), dict(top_p=0.7), dict(top_k=100, top_p=0.999)):
        got = ops.sample(x, u, temperature=T, **s)
        want = [R.sample(x[r], u[r], float(T[r]), s.get("top_k", 0), s.get("top_p", 1.0),
                         float(m[r]) if "min_p" in s else 0.0) for r in range(4)]
        assert got.tolist() == want
    assert ops.sample(x, u, min_p=1e-305).tolist() == ops.sample(x, u).tolist()
