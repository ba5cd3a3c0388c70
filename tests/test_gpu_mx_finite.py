"""The products' tests again under a comparison that takes no NaN for right, and outputs that start as NaN."""

import numpy as np
import pytest
import torch

import _mx
import test_gpu_mx as base
from _mx_check import check_product
from test_gpu_mx import (  # noqa: F401
    SHAPES, activations, dev, host, ops, test_gather_many_rows, test_gather_many_tiles, test_gather_promise_broken_is_contained,
    test_gather_qmm, test_mx_matmul, test_mx_matmul_grouped, test_product_forms, test_product_in_a_graph,
    test_product_rows_that_are_not_numbers, test_products_on_another_stream, test_quantized_matmul, test_wide_products,
    test_widths_of_many_rows)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def finite(monkeypatch):
    monkeypatch.setattr(base, "check_product", check_product)


@pytest.mark.parametrize("kind", ["bf16", "f16", "mx"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_every_output_is_written(ops, M, N, K, kind):  # noqa: F811
    rng = np.random.default_rng(M + N + K)
    w, s, wv = _mx.random_weights(rng, (N, K))
    # a margin of NaN behind the result as well: nothing is written past it
    buf = torch.full((M * N + 64,), float("nan"), dtype=torch.float16 if kind == "f16" else torch.bfloat16,
                     device="cuda")
    out = buf[:M * N].view(M, N)
    if kind == "mx":
        xq, xs, xv = _mx.random_weights(rng, (M, K), 8, 1.0)
        ops.mx_matmul(dev(xq), dev(xs), dev(w), dev(s), out=out)
    else:
        x = activations(rng, M, K, kind)
        xv = host(x)
        ops.quantized_matmul(x, dev(w), dev(s), None, group_size=32, bits=4, mode="mxfp4", out=out)
    check_product(out, xv, wv, kind == "f16")
    assert buf[M * N:].isnan().all()
