"""Grouped mxfp4 products of a few rows over many experts, where every row is an item of its own (at most 32
rows, four experts or more to a row): one decoded token's experts."""

import functools

import numpy as np
import pytest
import torch

import _mx
from _mx_check import check_product

pytestmark = pytest.mark.gpu

# rows, experts, N, K: odd widths and heights, up to 10 k-blocks of 256, one tile to many of a block
SHAPES = [(1, 4, 300, 1056), (1, 64, 8, 32), (10, 512, 264, 288), (3, 12, 130, 2080), (8, 40, 640, 2560),
          (32, 128, 257, 512), (20, 100, 1000, 1312), (32, 128, 2600, 1280)]
KINDS = ["bf16", "f16", "mx"]


@functools.lru_cache(maxsize=1)
def bank(E, N, K):
    rng = np.random.default_rng(E + N + K)
    w = rng.integers(0, 1 << 32, size=(E, N, K // 8), dtype=np.uint32).view(np.int32)
    s = rng.integers(116, 124, size=(E, N, K // 32)).astype(np.uint8)
    values = functools.lru_cache(maxsize=None)(lambda e: _mx.values(w[e], s[e], 4))
    return torch.from_numpy(w).cuda(), torch.from_numpy(s).cuda(), values


def call(kind, x, w, s, ids, src, sort):
    from mlxturbo_b200 import ops

    if kind == "mx":
        return ops.mx_matmul(*x, w, s, rhs_indices=ids, lhs_indices=src, sorted_indices=sort)
    y = ops.gather_qmm(x.unsqueeze(1), w, s, None, lhs_indices=src, rhs_indices=ids, group_size=32, bits=4,
                       mode="mxfp4", sorted_indices=sort)
    return y.squeeze(1)


@pytest.mark.parametrize("rows,E,N,K", SHAPES)
@pytest.mark.parametrize("kind", KINDS)
def test_each_row_its_own_expert(rows, E, N, K, kind):
    from mlxturbo_b200 import ops

    rng = np.random.default_rng(rows + E + N + K + len(kind))
    w, s, values = bank(E, N, K)
    T = rows // 2 + 1
    for ids in (rng.permutation(E)[:rows],                   # all different
                rng.integers(-3, E + 4, size=rows),          # some outside, some met twice
                np.full(rows, E - 1),                        # one expert
                np.where(np.arange(rows) % 2, -1, E)):       # none
        for sort in (False, True):
            i = np.sort(ids) if sort else ids
            for lhs in (None, rng.integers(0, T, size=rows)):
                M = rows if lhs is None else T
                if kind == "mx":
                    xq, xs, xv = _mx.random_weights(rng, (M, K), 8, 1.0)
                    x = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
                else:
                    x = torch.from_numpy(rng.normal(size=(M, K))).to(
                        torch.bfloat16 if kind == "bf16" else torch.float16).cuda()
                    xv = x.double().cpu().numpy()
                i32 = torch.from_numpy(i.astype(np.int32)).cuda()
                l32 = None if lhs is None else torch.from_numpy(lhs.astype(np.int32)).cuda()
                y = call(kind, x, w, s, i32, l32, sort)
                assert y.shape == (rows, N)
                for r in range(rows):
                    if 0 <= i[r] < E:
                        row = r if lhs is None else lhs[r]
                        check_product(y[r:r + 1], xv[row:row + 1], values(int(i[r])), kind == "f16", f"row {r}")
                    else:
                        assert (y[r] == 0).all()
                same = torch.stack([(call(kind, x, w, s, i32, l32, sort) == y).all() for _ in range(20)])
                assert same.all()
    assert ops.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_are_not_numbers_stay_alone(kind):
    """A NaN or an infinity gives its own row NaN; the rows of other items are untouched."""
    rng = np.random.default_rng(3)
    rows, E, N, K = 12, 64, 400, 800
    w, s, values = bank(E, N, K)
    ids = rng.permutation(E)[:rows].astype(np.int32)
    if kind == "mx":
        xq, xs, xv = _mx.random_weights(rng, (rows, K), 8, 1.0)
        xs[4, 7] = 255
        x = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
    else:
        x = torch.from_numpy(rng.normal(size=(rows, K))).to(torch.bfloat16 if kind == "bf16" else torch.float16).cuda()
        xv = x.double().cpu().numpy()
        x[4, 300] = float("nan") if kind == "bf16" else float("inf")
    y = call(kind, x, w, s, torch.from_numpy(ids).cuda(), None, False)
    assert not y[4].isfinite().any()
    for r in range(rows):
        if r != 4:
            check_product(y[r:r + 1], xv[r:r + 1], values(int(ids[r])), kind == "f16", f"row {r}")
