"""Products at the ends of the range of bf16 and of the scale bytes, in small products and large ones."""

import numpy as np
import pytest
import torch

import _mx
from _mx_check import check_product

pytestmark = pytest.mark.gpu

MX = dict(group_size=32, bits=4, mode="mxfp4")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def small_weights(rng, N, K):
    """mxfp4 weights of at most 6 * 2^-12, so that the sums stay in the range of bf16."""
    w, s, _ = _mx.random_weights(rng, (N, K))
    s = rng.integers(105, 116, size=s.shape).astype(np.uint8)
    return w, s, _mx.values(w, s, 4)


@pytest.mark.parametrize("M,N", [(1, 72), (2, 72), (7, 72), (20, 72), (40, 72), (300, 72), (300, 4900)])
def test_largest_bf16_values(M, N):
    """Finite magnitudes of 2^127 and above are numbers, whatever the other rows of the call."""
    from mlxturbo_b200 import ops

    rng = np.random.default_rng(M)
    K = 288
    w, s, wv = small_weights(rng, N, K)
    x = rng.normal(size=(M, K))
    x[:, 32:64] *= 2.0 ** 125                             # a block up to about 2^127
    x[0, 40], x[0, 41], x[0, 63] = 1.5 * 2.0 ** 127, -(2.0 - 2.0 ** -7) * 2.0 ** 127, 2.0 ** 127
    x[-1, 64:96] = rng.choice([-1.0, 1.0], size=32) * 2.0 ** 127 * (1 + rng.integers(0, 128, size=32) / 128)
    x = dev(np.clip(x, -(2.0 - 2.0 ** -7) * 2.0 ** 127, (2.0 - 2.0 ** -7) * 2.0 ** 127)).bfloat16()
    assert x.isfinite().all() and (x.abs() >= 2.0 ** 127).any()
    y = ops.quantized_matmul(x, dev(w), dev(s), None, **MX)
    check_product(y, x.double().cpu().numpy(), wv, False)


@pytest.mark.parametrize("M", [1, 2, 7, 20, 300])
@pytest.mark.parametrize("byte", [245, 246, 247, 250, 254])
def test_largest_scale_bytes(M, byte):
    """mxfp8 blocks whose values are below 2^128 are numbers, all zeros included."""
    from mlxturbo_b200 import ops

    rng = np.random.default_rng(M + byte)
    N, K = 40, 160
    w, s, wv = small_weights(rng, N, K)
    xq, xs, _ = _mx.random_weights(rng, (M, K), 8, 1.0)
    code = xq.view(np.uint8).reshape(M, K).copy()
    # exponent fields so that |code| * 2^(byte - 127) < 2^128 (a code of field f is below 2^(f - 6))
    code[:, 32:64] = rng.integers(0, min(127, 8 * max(1, 262 - byte)), size=(M, 32)) | (rng.integers(0, 2, size=(M, 32)) << 7)
    code[0, 96:128] = 0
    xs[:, 1] = byte
    xs[0, 3] = byte
    xq = code.view("<u4").view(np.int32)
    xv = _mx.values(xq, xs, 8)
    assert np.isfinite(xv).all() and np.abs(xv).max() < 2.0 ** 128
    y = ops.mx_matmul(dev(xq), dev(xs), dev(w), dev(s))
    check_product(y, xv, wv, False)


@pytest.mark.parametrize("M", [2, 7, 20, 300])
def test_infinite_stays_infinite(M):
    """An infinity, or an mxfp8 value of 2^128 and above, still gives its row no finite number."""
    from mlxturbo_b200 import ops

    rng = np.random.default_rng(M)
    N, K = 40, 160
    w, s, wv = small_weights(rng, N, K)
    x = dev(rng.normal(size=(M, K))).bfloat16()
    x[0, 70] = float("inf")
    x[0, 71] = (2.0 - 2.0 ** -7) * 2.0 ** 127
    y = ops.quantized_matmul(x, dev(w), dev(s), None, **MX)
    assert not y[0].isfinite().any()
    check_product(y[1:], x[1:].double().cpu().numpy(), wv, False)
    xq, xs, xv = _mx.random_weights(rng, (M, K), 8, 1.0)
    xs[0, 2] = 255
    y = ops.mx_matmul(dev(xq), dev(xs), dev(w), dev(s))
    assert y[0].isnan().all()
    check_product(y[1:], xv[1:], wv, False)


@pytest.mark.parametrize("M,N,small", [(1, 40, True), (2, 40, True), (7, 40, True), (20, 40, True), (300, 40, True),
                                       (300, 4900, False)])
@pytest.mark.parametrize("kind", ["bf16", "mx"])
def test_smallest_values(M, N, small, kind):
    """Blocks down to the subnormals against weights of up to 2^100: within 2^-126 a value in small products."""
    from mlxturbo_b200 import ops

    rng = np.random.default_rng(M)
    K = 192
    w, s, _ = _mx.random_weights(rng, (N, K))
    s = rng.integers(200, 225, size=s.shape).astype(np.uint8)
    wv = _mx.values(w, s, 4)
    if kind == "bf16":
        x = rng.normal(size=(M, K)) * np.repeat(2.0 ** rng.integers(-132, -95, size=(M, K // 32)), 32, axis=-1)
        x = dev(x).bfloat16()
        xv = x.double().cpu().numpy()
        y = ops.quantized_matmul(x, dev(w), dev(s), None, **MX)
    else:
        xq, xs, _ = _mx.random_weights(rng, (M, K), 8, 1.0)
        xs = rng.integers(0, 30, size=xs.shape).astype(np.uint8)
        xv = _mx.values(xq, xs, 8)
        y = ops.mx_matmul(dev(xq), dev(xs), dev(w), dev(s))
    ref = xv @ wv.T
    held = 2.0 ** -126 * np.abs(wv).sum(-1) if small else 0.0
    bound = _mx.product_bound(xv, wv, ref, False) + held
    assert (np.abs(y.double().cpu().numpy() - ref) <= bound).all()
