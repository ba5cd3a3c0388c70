"""Row tables of grouped mxfp4 products whose ids were promised to be sorted."""

import numpy as np
import pytest
import torch

import _mx
from _mx_check import check_product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["random", "descending", "ends"])
@pytest.mark.parametrize("rows", [5000, 60000])
def test_promise_broken_over_many_experts(rows, order):
    """Tables of far more items than rows allow: cut off within their arrays, and the next call is right."""
    from mlxturbo_b200 import ops

    rng = np.random.default_rng(rows)
    E, N, K = 2000, 16, 32
    w, s, wv = _mx.random_weights(rng, (E, N, K))
    w, s = torch.from_numpy(w).cuda(), torch.from_numpy(s).cuda()
    ids = rng.integers(-3, E + 3, size=rows).astype(np.int32)
    if order == "descending":
        ids = np.sort(ids)[::-1].copy()
    elif order == "ends":
        ids = np.where(np.arange(rows) % 2, 0, E - 1).astype(np.int32)
    x = torch.from_numpy(rng.normal(size=(64, K))).bfloat16().cuda()
    src = rng.integers(0, 64, size=rows).astype(np.int32)
    kw = dict(lhs_indices=torch.from_numpy(src).cuda(), group_size=32, bits=4, mode="mxfp4")
    ops.gather_qmm(x[:, None], w, s, None, rhs_indices=torch.from_numpy(ids).cuda(), sorted_indices=True, **kw)
    assert ops.device_error() == 0
    at = np.argsort(ids, kind="stable")
    kw["lhs_indices"] = torch.from_numpy(src[at]).cuda()
    y = ops.gather_qmm(x[:, None], w, s, None, rhs_indices=torch.from_numpy(ids[at]).cuda(), sorted_indices=True, **kw)
    assert ops.device_error() == 0
    ids, xv = ids[at], x.double().cpu().numpy()[src[at]]
    for e in np.unique(ids)[:: 1 if order == "ends" else 40]:
        r = np.flatnonzero(ids == e)
        rows_e = y[torch.from_numpy(r).cuda(), 0]
        if 0 <= e < E:
            check_product(rows_e, xv[r], wv[int(e)], False, f"expert {e}")
        else:
            assert (rows_e == 0).all()
