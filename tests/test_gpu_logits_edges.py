"""Rows of logits where a border, a list or a sum lies at the edge of what 32 or 64 bits tell apart."""

import math

import numpy as np
import pytest
import torch

import _logits as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture
def ops():
    from mlxturbo_b200 import ops

    return ops


def uniform(seed, *shape):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [3, 4099, 70001])
def test_min_p_border_around_zero(ops, V, dtype):
    """A largest logit of 0, or a border there: keys of 32 bits are dense around it, weights alike."""
    g = torch.Generator().manual_seed(V)
    x = -0.01 - torch.rand((8, V), generator=g) * 6
    for at in (-4.0, -5.0):  # no logit where its last bit decides
        x[(x - at).abs() < 0.05] = -4.5
    x[0] = 0.0
    x[1, ::3] = 0.0  # equal largest ones
    x[2, V // 2] = -0.0
    x[3, V - 1], x[3, 1] = 0.0, -1e-20 if dtype == torch.float32 else -0.5  # weighs 1 in 64 bits too
    x[4, 0] = 1e-20 if dtype == torch.float32 else 1e-7
    x[5, 1] = 5.0
    x[6, 1], x[6, 2] = 4.0, 0.25
    x[7] = torch.finfo(dtype).min
    x, u = x.to(dtype).cuda(), uniform(1, 8)
    T = torch.tensor([1.0, 0.5, 2.0, 1.0, 1e-6, 3e38, math.inf, 1e30]).cuda()
    for s in (dict(min_p=1.0), dict(min_p=math.exp(-5.0)), dict(temperature=0.5, min_p=math.exp(-8.0)),
              dict(top_k=2, min_p=1.0), dict(top_p=0.5, min_p=1.0), dict(temperature=T, min_p=1.0),
              dict(temperature=T, min_p=torch.full((8,), 3.0).cuda())):
        got = ops.sample(x, u, **s)
        t = s.get("temperature", 1.0)
        m = s["min_p"]
        # Exponentials in 64 bits agree to a few roundings: with |t| = |x - max| log2(e) / T below 8 here, c, the offset
        # and the difference are off by 2^-53 each of at most 8, t so by 2^-48, the weight by ln 2 times that and the
        # polynomial's 3e-15: below 2^-47.  A weight that near to min_p (fp16 has -1.0 = 4 - 5) may fall to either side.
        wants = [[R.sample(x[r], u[r], float(t[r]) if torch.is_tensor(t) else t, s.get("top_k", 0), s.get("top_p", 1.0),
                           (float(m[r]) if torch.is_tensor(m) else m) * (1 + side * 2.0 ** -47)) for side in (-1, 1)]
                 for r in range(8)]
        assert all(i in w for i, w in zip(got.tolist(), wants)), (s, got.tolist(), wants)


@pytest.mark.parametrize("B,n", [(2, 33), (3, 1500)])
def test_speculative_long_drafts(ops, B, n):
    """More positions than a warp has lanes, a draft that ends behind them, one that ends there."""
    V = 8
    g = torch.Generator().manual_seed(n)
    logits = torch.randn((B, n + 1, V), generator=g).cuda()
    draft = logits[:, :n].clone()  # every token stands ...
    ids = torch.randint(0, V, (B, n), generator=g).cuda()
    u = uniform(2, B, n + 1)
    ids[0, n - 1] = -1
    draft[1, n - 1] = -20.0
    draft[1, n - 1, ids[1, n - 1]] = 20.0  # ... but this one, nearly always
    u[1, n - 1] = 0.999
    tokens, accepted = ops.speculative_sample(logits, draft, ids, u)
    for b in range(B):
        want, j = R.speculative(logits[b], draft[b], ids[b], u[b])
        assert tokens[b].tolist() == want and int(accepted[b]) == j
    assert accepted.tolist()[:2] == [n - 1, n - 1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 5003, 120001])
def test_numbers_near_zero(ops, V, dtype):
    """u = 0, or far below 2^-53, asks for tokens that weigh nothing beside the sum: the first id that is kept."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn((12, V), generator=g) * 3
    for r in range(12):
        x[r, torch.randperm(V, generator=g)[:5]] = 60.0 - r
    x[6:, :4] = torch.tensor([-9.0, 12.0, 9.0, 20.0])
    x = x.to(dtype).cuda()
    u = torch.tensor([0.0, 0.0, 1e-30, 1e-38, 1e-20, 1e-12] * 2).cuda()
    for s in (dict(top_k=2), dict(top_k=6), dict(temperature=0.5, top_k=30), dict(temperature=0.3, top_k=20, top_p=0.999),
              dict(top_k=39, min_p=1e-30), dict(temperature=0.7, top_k=300), dict(min_p=1e-25), dict(min_p=1e-9),
              dict(temperature=0.6), dict(temperature=2.0)):
        if s.get("top_k", 0) >= V:
            continue
        want = [R.sample(x[r], u[r], s.get("temperature", 1.0), s.get("top_k", 0), s.get("top_p", 1.0), s.get("min_p", 0.0))
                for r in range(12)]
        assert ops.sample(x, u, **s).tolist() == want, s


def _far_tokens(V, seed, first):
    """A row of five tokens that weigh 1, 4000 that weigh 1e-10 each, and id 3 with logit `first`; k and top-p keep
    most of the 4000."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((V,), -60.0)
    at = V // 2 + torch.randperm(V // 2, generator=g)[:4005]
    x[at] = -23.5 + torch.rand(4005, generator=g)
    x[at[:5]] = 0.0
    x[3] = first
    return x


def test_draws_finer_than_the_bins(ops):
    """Masses that bins hold in whole parts of 2^-40: a draw that falls between a token's weight and its rounding."""
    V, k, p = 120001, 4500, 1 - 1e-9
    unit = 2.0 ** -40
    rows, u = [], []
    for i in range(40):
        first = -22.6 - i / 400
        x = _far_tokens(V, i, first)
        own = math.exp(float(x[3]))
        whole = round(own / unit)
        l = R.values(x)
        w = R.weights(l, 1.0)[R.order(l)[:k]]
        mass = w.cumsum()
        total = mass[int((mass - w < p * mass[-1]).sum()) - 1]
        rows.append(x)
        u.append((own + whole * unit) / 2 / total)  # between the weight and the whole number
    x, u = torch.stack(rows).cuda(), torch.tensor(u, dtype=torch.float32).cuda()
    want = [R.sample(x[r], u[r], 1.0, k, p) for r in range(40)]
    assert 5 < sum(i == 3 for i in want) < 35  # either side
    assert ops.sample(x, u, top_k=k, top_p=p).tolist() == want


def test_borders_finer_than_the_bins(ops):
    """A border of top-p that falls within the rounding of the thousands of masses above it: id 3 is kept or not."""
    V, k = 120001, 4500
    u = torch.zeros(24, device="cuda")
    seen = set()
    for seed in range(12):
        x = _far_tokens(V, seed, -23.3)
        l = R.values(x)
        o = R.order(l)[:k]
        mass = R.weights(l, 1.0)[o].cumsum()
        before = mass[o.tolist().index(3) - 1]
        for side in (-1, 1):
            p = float((before + side * 2.0 ** -40) / mass[-1])
            want = R.sample(x, 0.0, 1.0, k, p)
            seen.add(want == 3)
            got = ops.sample(x.cuda().expand(24, -1), u, top_k=k, top_p=p)
            assert got.tolist() == [want] * 24, (seed, side)
    assert seen == {True, False}


@pytest.mark.parametrize("dtype", DTYPES)
def test_first_and_last_draws_of_open_rows(ops, dtype):
    """u = 0 and the last number below 1 where bins hold the masses, with and without min-p."""
    V = 60013
    g = torch.Generator().manual_seed(1)
    x = (torch.randn((16, V), generator=g) * 1.8).to(dtype).cuda()
    u = torch.tensor([0.0, 1e-30, 1e-9, 1 - 2 ** -24] * 4).cuda()
    for s in (dict(top_p=0.95), dict(top_p=0.5, temperature=1.5), dict(top_k=3000, top_p=0.9), dict(top_k=20000),
              dict(top_p=0.9, min_p=1e-4)):
        want = [R.sample(x[r], u[r], s.get("temperature", 1.0), s.get("top_k", 0), s.get("top_p", 1.0), s.get("min_p", 0.0))
                for r in range(16)]
        assert ops.sample(x, u, **s).tolist() == want, s


def test_border_searched_at_a_token_s_end(ops):
    """top-p whose target is the mass up to a token to the last bits, where the border is searched by passes (a
    vocabulary of 262144): the passes cut their sums in different ways, and none may lose the border."""
    V, rows = 262144, 12
    u = torch.full((rows,), 0.5, device="cuda")
    for seed in range(10):
        x = (torch.randn(V, generator=torch.Generator().manual_seed(seed)) * 1.5).cuda()
        l = R.values(x)
        w, o = R.weights(l, 1.0), R.order(l)
        mass = w[o].cumsum()
        rank = np.empty(V, np.int64)
        rank[o] = np.arange(V)
        for depth in (3.5, 5.5, 8.0):  # where the first pass cuts
            n = int((l >= np.float32(l.max()) - np.float32(depth)).sum())
            want = set()
            for kept in (n - 1, n, n + 1):  # which of them: the last bits
                cum = (w * (rank < kept)).cumsum()
                want.add(int((cum > 0.5 * cum[-1]).argmax()))
            for bits in range(-40, 41):
                p = float(mass[n - 1] / mass[-1]) * (1 + bits * 2.0 ** -52)
                got = ops.sample(x.expand(rows, -1), u, top_p=p)
                assert set(got.tolist()) <= want, (seed, depth, bits)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_of_any_size(ops, dtype):
    """Stretches of a row that a mask fills with one huge number, at every temperature."""
    V = 70003
    g = torch.Generator().manual_seed(5)
    x = torch.randn((6, V), generator=g) * 2
    hide = torch.rand((6, V), generator=g) < 0.7
    hide[:, 50:V // 2] = True
    u = uniform(6, 6)
    for size in (1e4, 1e9, 1e10, 3e20, 1e30, 2.9e38, 3.3e38):
        if size > torch.finfo(dtype).max:
            continue
        y = x.masked_fill(hide, -size).to(dtype).cuda()
        ids = y[:, :2].argmax(-1)[:, None]
        for T in (0.3, 1.0, 2.0, 4.0):
            for s in (dict(), dict(top_p=0.9), dict(top_k=300, top_p=0.9)):
                want = [R.sample(y[r], u[r], T, s.get("top_k", 0), s.get("top_p", 1.0)) for r in range(6)]
                assert ops.sample(y, u, temperature=T, **s).tolist() == want, (size, T, s)
            lse = ops.topk(y, 3, logsumexp=True, temperature=T)[2]
            for r in range(6):
                want = R.logsumexp(y[r], T)
                assert abs(float(lse[r]) - want) <= 1e-5 + 2 ** -24 * abs(want)
            tokens, accepted = ops.speculative_sample(y.view(3, 2, V), y.view(3, 2, V)[:, 1:], ids[::2], u.view(3, 2),
                                                      temperature=T)
            for b in range(3):
                want, j = R.speculative(y[2 * b:2 * b + 2], y[2 * b + 1:2 * b + 2], ids[2 * b], u[2 * b:2 * b + 2], T)
                assert tokens[b].tolist() == want and int(accepted[b]) == j


def test_topk_of_more_than_a_row(ops):
    """Refused before outputs of that size are asked for."""
    x = torch.randn((3, 50), device="cuda")
    before = torch.cuda.memory_allocated()
    for k in (51, 2 ** 31, 2 ** 40, 2 ** 62):
        with pytest.raises(ValueError, match="not in"):
            ops.topk(x, k, logsumexp=True)
    assert torch.cuda.memory_allocated() == before
