"""The comparison the product tests rest on: right results pass, and a NaN, an infinity or a moved value does not."""

import numpy as np
import pytest
import torch

import _mx
from _mx_check import check_product


@pytest.mark.parametrize("wrong", [None, float("nan"), float("inf"), 1.5])
def test_check_product(wrong):
    rng = np.random.default_rng(0)
    _, _, w = _mx.random_weights(rng, (24, 96))
    x = rng.normal(size=(5, 96))
    y = torch.from_numpy(x @ w.T).bfloat16()
    if wrong is None:
        check_product(y, x, w, False)
        return
    y[3, 7] = wrong if wrong != 1.5 else y[3, 7] * 1.5 + 1
    with pytest.raises(AssertionError):
        check_product(y, x, w, False)
    with pytest.raises(AssertionError):
        check_product(torch.full_like(y, wrong), x, w, False)
