"""Comparison of products with their value in 64 bits that takes no NaN for right."""

import numpy as np

import _mx


def check_product(y, x, w, f16, what=""):
    """y [M, N] (torch) against x [M, K] @ w [N, K]^T (numpy, 64 bits): finite and within the bound everywhere."""
    ref = x @ w.T
    got = y.double().cpu().numpy()
    assert np.isfinite(ref).all(), f"{what}: the reference is to be finite"
    right = np.abs(got - ref) <= _mx.product_bound(x, w, ref, f16)  # False for a NaN
    assert right.all(), f"{what}: {(~right).sum()} of {right.size} off, {np.isnan(got).sum()} of them not a number"
