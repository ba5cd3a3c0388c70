"""Rows of logits where a border, a list or a sum lies at the edge of what 32 or 64 bits tell apart."""

import math

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
