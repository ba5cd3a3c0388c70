"""Microscaled (MX) operators against their definition in 64 bits."""

import numpy as np
import pytest
import torch

import _mx

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from mlxturbo_b200 import ops as o

    return o


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(DT[dtype])


def host(t):
    return t.double().cpu().numpy()


# --------------------------------------------------------------------------
# quantize / dequantize
# --------------------------------------------------------------------------

def wide_values(rng, shape, dtype):
    """Blocks of very different sizes, ties of both grids, zeros and subnormals."""
    v = rng.normal(size=shape) * 2.0 ** rng.integers(-10, 10, size=(*shape[:-1], 1))
    flat = v.reshape(-1, 32)
    flat[::7] = rng.choice([0.0, -0.0, 0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5.0, 6.0, 7.5], size=flat[::7].shape)
    flat[3::11] = 0.0
    flat[5::13] = rng.integers(-300, 300, size=flat[5::13].shape) * (2.0 ** -24 if dtype == "f16" else 2.0 ** -133)
    if dtype != "f16":
        flat[6::17] *= 2.0 ** 100
        flat[8::19] *= 2.0 ** -110
    return torch.from_numpy(v).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (7, 96), (33, 5120), (2, 5, 160), (1001, 32)])
def test_quantize_is_the_definition(ops, shape, bits, dtype):
    rng = np.random.default_rng(shape[-1] + bits)
    v = wide_values(rng, shape, dtype)
    code, scale = _mx.quantize(v.double().numpy(), bits)
    mode = "mxfp4" if bits == 4 else "mxfp8"
    wq, s = ops.quantize(v.cuda(), 32, bits, mode=mode)
    assert wq.dtype == torch.int32 and s.dtype == torch.uint8
    assert np.array_equal(s.cpu().numpy(), scale)
    assert np.array_equal(wq.cpu().numpy(), _mx.pack(code, bits))
    for out in ("bf16", "f16", "f32"):
        got = ops.dequantize(wq, s, None, 32, bits, mode=mode, dtype=DT[out])
        want = torch.from_numpy(_mx.values(wq, s, bits)).float().to(DT[out])
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_blocks_that_are_not_numbers(ops, bits):
    v = torch.ones(1, 160)
    v[0, 5], v[0, 40], v[0, 70] = float("nan"), float("inf"), float("-inf")
    wq, s = ops.quantize(v.cuda(), 32, bits, mode=f"mxfp{bits}")
    assert s.cpu().tolist() == [[255, 255, 255, 127 - (2 if bits == 4 else 8), 127 - (2 if bits == 4 else 8)]]
    got = ops.dequantize(wq, s, None, 32, bits, mode=f"mxfp{bits}", dtype=torch.float32).cpu()
    assert got[0, :96].isnan().all() and (got[0, 96:] == 1).all()


def test_every_code_and_scale(ops):
    """All 256 scale bytes against every code, to all three types."""
    scale = np.arange(256, dtype=np.uint8).reshape(256, 1)
    for bits, code in ((4, np.tile(np.arange(16, dtype=np.uint8), 2)), (8, None)):
        rows = [code] if bits == 4 else np.arange(256, dtype=np.uint8).reshape(8, 32)
        for c in rows:
            w = _mx.pack(np.broadcast_to(c, (256, 32)), bits)
            want = torch.from_numpy(_mx.values(w, scale, bits)).float()
            for out in DT.values():
                got = ops.dequantize(dev(w), dev(scale), None, 32, bits, mode=f"mxfp{bits}", dtype=out)
                assert torch.equal(got.cpu().nan_to_num(12345.0), want.to(out).nan_to_num(12345.0))


def test_quantize_takes_strided_and_empty_values(ops):
    v = torch.randn(40, 256, device="cuda", dtype=torch.bfloat16)
    a = ops.quantize(v[::3, 64:192], 32, 4, mode="mxfp4")
    b = ops.quantize(v[::3, 64:192].contiguous(), 32, 4, mode="mxfp4")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a = ops.quantize(v.t()[:, :32], 32, 8, mode="mxfp8")
    b = ops.quantize(v.t()[:, :32].contiguous(), 32, 8, mode="mxfp8")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    w, s = ops.quantize(v[:0], 32, 4, mode="mxfp4")
    assert w.shape == (0, 32) and s.shape == (0, 8)
    assert ops.dequantize(w, s, None, 32, 4, mode="mxfp4").shape == (0, 256)


# --------------------------------------------------------------------------
# norm
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,K", [(1, 32), (5, 64), (1, 5120), (9, 2048), (300, 640), (3, 8192), (2, 12320),
                                    (2, 16384), (3, 32768), (2, 40960)])
def test_norm(ops, rows, K, residual, dtype):
    rng = np.random.default_rng(rows * K)
    x, r = dev(rng.normal(size=(rows, K)), dtype), dev(3 * rng.normal(size=(rows, K)), dtype)
    g = dev(1 + 0.2 * rng.normal(size=K), dtype)
    xq, xs, h = ops.rms_norm_quantize(x, g, 1e-5, residual=r if residual else None)
    s = x.float() + (r.float() if residual else 0)
    if residual:
        assert torch.equal(h, s.to(DT[dtype]))
    else:
        assert h is None
    s64 = host(x) + (host(r) if residual else 0)
    y = s64 / np.sqrt((s64 ** 2).mean(-1, keepdims=True) + 1e-5) * host(g)
    code, scale = _mx.quantize(y, 8)
    want = _mx.values(_mx.pack(code, 8), scale, 8)
    got = _mx.values(xq, xs, 8)
    # fp32 arithmetic moves a value by at most about 2^-20 of itself, so only one
    # that lies this near the middle between two codes may round the other way,
    # and only a block whose largest value lies this near a power of two may take
    # the neighbouring scale: one code step (up to 1/7 of the value, or 2^-9 of
    # the larger scale below the smallest normal code) either way.
    step = np.maximum(np.abs(want) / 7, np.repeat(np.ldexp(1.0, scale.astype(int) - 127 - 9), 32, axis=-1) * 2)
    assert (np.abs(got - want) <= step).all()
    assert (got != want).mean() <= 1e-3
    assert (np.abs(xs.cpu().numpy().astype(int) - scale.astype(int)) <= 1).all()


def test_norm_edge_rows(ops):
    """A zero row, a row with a NaN, one with an infinity, and one whose squares are tiny."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    x[1], x[2], x[3] = 1, 1, 2.0 ** -60
    x[1, 3], x[2, 40] = float("nan"), float("inf")
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    xq, xs, h = ops.rms_norm_quantize(x, g, 1e-6, residual=torch.zeros_like(x))
    v = _mx.values(xq, xs, 8)
    assert (v[0] == 0).all() and np.isnan(v[1]).all()
    # infinity: the mean is infinite, finite values become 0 and the infinite one NaN, with its block
    assert (v[2, :32] == 0).all() and np.isnan(v[2, 32:]).all()
    # e4m3 is off by at most 1/16 of the value
    want = 2.0 ** -60 / np.sqrt(2.0 ** -120 + 1e-6)
    assert np.allclose(v[3], want, rtol=1 / 16)
    assert torch.equal(h.nan_to_num(7.0), x.nan_to_num(7.0))


def test_norm_leading_axes_and_strides(ops):
    x = torch.randn(2, 3, 256, device="cuda", dtype=torch.float16)
    g = torch.ones(256, device="cuda", dtype=torch.float16)
    xq, xs, h = ops.rms_norm_quantize(x.transpose(0, 1), g, residual=x.transpose(0, 1))
    assert xq.shape == (3, 2, 64) and xs.shape == (3, 2, 8) and h.shape == (3, 2, 256)
    a, b, _ = ops.rms_norm_quantize(x.transpose(0, 1).contiguous(), g, residual=x.transpose(0, 1).contiguous())
    assert torch.equal(xq, a) and torch.equal(xs, b)
    xq, xs, h = ops.rms_norm_quantize(x[:0], g, residual=x[:0])
    assert xq.shape == (0, 3, 64) and h.shape == (0, 3, 256)


# --------------------------------------------------------------------------
# products
# --------------------------------------------------------------------------

def check_product(y, x, w, f16, what=""):
    ref = x @ w.T
    bad = np.abs(host(y) - ref) > _mx.product_bound(x, w, ref, f16)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.abs(host(y) - ref)[bad].max()}"


def activations(rng, M, K, dtype):
    """Normal values with a few large outliers, as hidden states have."""
    x = rng.normal(size=(M, K))
    x[rng.random(size=x.shape) < 0.002] *= 50
    return dev(x, dtype)


SHAPES = [
    (1, 8, 32), (1, 1, 96), (3, 40, 160), (1, 128, 128), (1, 1024, 5120), (2, 300, 2048), (5, 1000, 640),
    (8, 257, 1024), (9, 384, 512), (16, 200, 2048), (17, 130, 256), (33, 128, 384), (64, 640, 2048), (65, 129, 128),
    (130, 512, 1664), (257, 384, 512), (300, 1000, 640), (513, 260, 1152), (40, 96, 224),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_quantized_matmul(ops, M, N, K, dtype):
    rng = np.random.default_rng(M + 10 * N + 100 * K)
    w, s, wv = _mx.random_weights(rng, (N, K))
    x = activations(rng, M, K, dtype)
    y = ops.quantized_matmul(x, dev(w), dev(s), None, group_size=32, bits=4, mode="mxfp4")
    assert y.shape == (M, N) and y.dtype == x.dtype
    check_product(y, host(x), wv, dtype == "f16")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_mx_matmul(ops, M, N, K, dtype):
    rng = np.random.default_rng(M + 10 * N + 100 * K + 1)
    w, s, wv = _mx.random_weights(rng, (N, K))
    xq, xs, xv = _mx.random_weights(rng, (M, K), 8, 1.0)
    y = ops.mx_matmul(dev(xq), dev(xs), dev(w), dev(s), dtype=DT[dtype])
    assert y.shape == (M, N) and y.dtype == DT[dtype]
    check_product(y, xv, wv, dtype == "f16")


@pytest.mark.parametrize("kind", ["bf16", "f16", "mx"])
@pytest.mark.parametrize("M,N,K", [(70, 300, 96), (193, 257, 4128), (400, 640, 2880), (90, 200, 8224), (17, 515, 2080),
                                   (65, 2500, 1056), (1000, 100, 32)])
def test_widths_of_many_rows(ops, M, N, K, kind):
    """Widths that end inside a k-block, parts of K that meet, rows of scale bytes on odd addresses."""
    rng = np.random.default_rng(M + N + K)
    w, s, wv = _mx.random_weights(rng, (N + 1, K))
    s[0] = s[3] = 255  # outside of the slice, and a row of its own
    w, s = dev(w)[1:], dev(s)[1:]
    if kind == "mx":
        xq, xs, xv = _mx.random_weights(rng, (M + 1, K), 8, 1.0)
        xs[0] = 255
        y = ops.mx_matmul(dev(xq)[1:], dev(xs)[1:], w, s)
        xv = xv[1:]
    else:
        x = activations(rng, M, K, kind)
        y = ops.quantized_matmul(x, w, s, None, group_size=32, bits=4, mode="mxfp4")
        xv = host(x)
    assert y[:, 2].isnan().all()
    keep = [n for n in range(N) if n != 2]
    check_product(y[:, keep], xv, wv[1:][keep], kind == "f16")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M", [1, 7, 40, 300])
def test_product_range(ops, M, dtype):
    """Scales far apart between blocks of one row, and inside a block."""
    rng = np.random.default_rng(M)
    K, N = 512, 200
    span = 6 if dtype == "f16" else 30
    w, s, _ = _mx.random_weights(rng, (N, K))
    s = (s.astype(int) + rng.integers(-span, span, size=s.shape)).clip(0, 254).astype(np.uint8)
    wv = _mx.values(w, s, 4)
    x = rng.normal(size=(M, K)) * 2.0 ** rng.integers(-span, span // 2, size=(M, K))
    x = dev(x, dtype)
    y = ops.quantized_matmul(x, dev(w), dev(s), None, group_size=32, bits=4, mode="mxfp4")
    ref = host(x) @ wv.T
    top = 65504 if dtype == "f16" else 3e38
    fine = np.abs(ref) < top
    bound = _mx.product_bound(host(x), wv, ref, dtype == "f16")
    assert (np.abs(host(y) - ref)[fine] <= bound[fine]).all()


def test_product_rows_that_are_not_numbers(ops):
    """A NaN stays in its row; a NaN weight block reaches every row of its column."""
    rng = np.random.default_rng(5)
    for M, N, K in ((3, 40, 160), (4, 256, 512), (70, 256, 512)):
        w, s, wv = _mx.random_weights(rng, (N, K))
        x = activations(rng, M, K, "bf16")
        x[1, 17], x[2, 33] = float("nan"), float("inf")
        s[7, 2] = 255
        y = ops.quantized_matmul(x, dev(w), dev(s), None, group_size=32, bits=4, mode="mxfp4")
        assert y[1].isnan().all() and not y[2].isfinite().any() and y[:, 7].isnan().all()
        keep = [i for i in range(M) if i not in (1, 2)]
        cols = [n for n in range(N) if n != 7]
        check_product(y[keep][:, cols], host(x)[keep], wv[cols], False)


def test_product_forms(ops):
    """Leading axes, strided activations, out, an empty batch, and equal bits on every call."""
    rng = np.random.default_rng(6)
    w, s, wv = _mx.random_weights(rng, (384, 256))
    x = activations(rng, 24, 512, "bf16")
    kw = dict(group_size=32, bits=4, mode="mxfp4")
    y = ops.quantized_matmul(x[:, ::2].reshape(2, 12, 256), dev(w), dev(s), None, **kw)
    assert y.shape == (2, 12, 384)
    check_product(y.reshape(24, 384), host(x[:, ::2]), wv, False)
    out = torch.empty(24, 384, dtype=torch.bfloat16, device="cuda")
    assert ops.quantized_matmul(x[:, ::2], dev(w), dev(s), None, out=out, **kw) is out
    assert torch.equal(out, y.reshape(24, 384))
    for _ in range(3):
        assert torch.equal(ops.quantized_matmul(x[:, ::2], dev(w), dev(s), None, **kw), out)
    assert ops.quantized_matmul(x[:0, :256], dev(w), dev(s), None, **kw).shape == (0, 384)
    # weights that are a view not aligned to 32 bytes
    big = torch.zeros(385 * 32 + 4, dtype=torch.int32, device="cuda")
    view = big[4:4 + 384 * 32].view(384, 32)
    view.copy_(dev(w))
    check_product(ops.quantized_matmul(x[:, ::2], view, dev(s), None, **kw), host(x[:, ::2]), wv, False)


@pytest.mark.parametrize("M,N,K", [(130, 512, 1664), (300, 1024, 1152), (64, 640, 2048), (5, 1000, 640), (20, 512, 2048)])
def test_products_repeat(ops, M, N, K):
    """Equal bits on every call: no sum, hand-over or buffer depends on timing."""
    rng = np.random.default_rng(M)
    w, s, _ = _mx.random_weights(rng, (N, K))
    xq, xs, _ = _mx.random_weights(rng, (M, K), 8, 1.0)
    w, s, xq, xs = dev(w), dev(s), dev(xq), dev(xs)
    x = {dt: activations(rng, M, K, dt) for dt in ("bf16", "f16")}
    calls = [lambda: ops.mx_matmul(xq, xs, w, s)] + [
        lambda v=v: ops.quantized_matmul(v, w, s, None, group_size=32, bits=4, mode="mxfp4") for v in x.values()]
    for call in calls:
        first = call()
        same = torch.stack([(call() == first).all() for _ in range(400)])
        assert same.all()
    assert ops.device_error() == 0


def test_products_on_another_stream(ops):
    rng = np.random.default_rng(7)
    w, s, wv = _mx.random_weights(rng, (512, 1024))
    w, s = dev(w), dev(s)
    xs = [activations(rng, 4, 1024, "bf16") for _ in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    ys = []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            for _ in range(20):
                y = ops.quantized_matmul(x, w, s, None, group_size=32, bits=4, mode="mxfp4")
            ys.append(y)
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        check_product(y, host(x), wv, False)


def test_product_in_a_graph(ops):
    rng = np.random.default_rng(8)
    w, s, wv = _mx.random_weights(rng, (640, 1024))
    w, s = dev(w), dev(s)
    x = activations(rng, 2, 1024, "bf16")
    kw = dict(group_size=32, bits=4, mode="mxfp4")
    ops.quantized_matmul(x, w, s, None, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.quantized_matmul(x, w, s, None, **kw)
    for _ in range(2):
        x.copy_(activations(rng, 2, 1024, "bf16"))
        g.replay()
        check_product(y, host(x), wv, False)


# --------------------------------------------------------------------------
# grouped by expert
# --------------------------------------------------------------------------

def check_grouped(y, x, ids, src, wv, f16):
    """Rows of each expert against its own matrix; rows without one are zero."""
    y = y.reshape(len(ids), -1)
    for e in np.unique(ids):
        at = np.flatnonzero(ids == e)
        if 0 <= e < wv.shape[0]:
            check_product(y[torch.from_numpy(at).cuda()], x[src[at]], wv[e], f16, f"expert {e}")
        else:
            assert (y[torch.from_numpy(at).cuda()] == 0).all()


IDS = {
    "spread": lambda rng, rows, E: rng.integers(0, E, size=rows),
    "one": lambda rng, rows, E: np.full(rows, E - 1),
    "skewed": lambda rng, rows, E: np.minimum(rng.zipf(1.5, size=rows) - 1, E - 1),
    "some_outside": lambda rng, rows, E: rng.integers(-2, E + 3, size=rows),
    "none_inside": lambda rng, rows, E: np.full(rows, E),
}


@pytest.mark.parametrize("kind", list(IDS))
@pytest.mark.parametrize("sort", [False, True])
@pytest.mark.parametrize("rows,E,N,K,dtype", [
    (1, 1, 8, 32, "bf16"), (10, 16, 128, 256, "bf16"), (10, 4, 72, 96, "f16"), (40, 8, 256, 512, "f16"),
    (64, 64, 200, 128, "bf16"), (300, 3, 130, 640, "bf16"), (700, 8, 256, 256, "f16"), (300, 3, 130, 672, "f16"),
])
def test_gather_qmm(ops, rows, E, N, K, dtype, sort, kind):
    rng = np.random.default_rng(rows + E + N + K)
    w, s, wv = _mx.random_weights(rng, (E, N, K))
    ids = IDS[kind](rng, rows, E).astype(np.int32)
    if sort:
        ids = np.sort(ids)
    T = max(1, rows // 2)
    src = rng.integers(0, T, size=rows).astype(np.int32)
    x = activations(rng, T, K, dtype)
    kw = dict(group_size=32, bits=4, mode="mxfp4", sorted_indices=sort)
    y = ops.gather_qmm(x.reshape(T, 1, K), dev(w), dev(s), None, lhs_indices=dev(src), rhs_indices=dev(ids), **kw)
    assert y.shape == (rows, 1, N) and y.dtype == x.dtype
    check_grouped(y, host(x), ids, src, wv, dtype == "f16")
    # without lhs_indices: row r of x
    xr = activations(rng, rows, K, dtype)
    y = ops.gather_qmm(xr.reshape(rows, 1, K), dev(w), dev(s), None, rhs_indices=dev(ids), **kw)
    check_grouped(y, host(xr), ids, np.arange(rows), wv, dtype == "f16")


@pytest.mark.parametrize("sort", [False, True])
@pytest.mark.parametrize("rows,E,N,K", [(10, 16, 128, 256), (90, 8, 72, 96), (500, 4, 256, 384), (500, 4, 136, 1056)])
def test_mx_matmul_grouped(ops, rows, E, N, K, sort):
    rng = np.random.default_rng(rows)
    w, s, wv = _mx.random_weights(rng, (E, N, K))
    ids = rng.integers(0, E, size=rows).astype(np.int32)
    ids = np.sort(ids) if sort else ids
    xq, xs, xv = _mx.random_weights(rng, (rows, K), 8, 1.0)
    y = ops.mx_matmul(dev(xq), dev(xs), dev(w), dev(s), rhs_indices=dev(ids), sorted_indices=sort)
    check_grouped(y, xv, ids, np.arange(rows), wv, False)
    src = rng.integers(0, rows, size=rows).astype(np.int32)
    y = ops.mx_matmul(dev(xq), dev(xs), dev(w), dev(s), lhs_indices=dev(src), rhs_indices=dev(ids),
                      sorted_indices=sort, dtype=torch.float16)
    check_grouped(y, xv, ids, src, wv, True)


def test_gather_many_rows(ops):
    """Past the one-launch sort (16384 rows), ids in token order."""
    rng = np.random.default_rng(9)
    rows, E, N, K = 17001, 12, 64, 128
    w, s, wv = _mx.random_weights(rng, (E, N, K))
    ids = rng.integers(-1, E + 1, size=rows).astype(np.int32)
    x = activations(rng, rows, K, "bf16")
    y = ops.gather_qmm(x.reshape(rows, 1, K), dev(w), dev(s), None, rhs_indices=dev(ids), group_size=32, bits=4,
                       mode="mxfp4")
    check_grouped(y, host(x), ids, np.arange(rows), wv, False)


@pytest.mark.parametrize("rows,E,N,K", [(100, 60, 2048, 512), (60, 40, 1920, 256), (90, 30, 1536, 768),
                                        (20, 100, 2048, 2560)])
def test_gather_many_tiles(ops, rows, E, N, K):
    """Several tiles and several experts to a block."""
    rng = np.random.default_rng(rows)
    w = rng.integers(0, 1 << 32, size=(E, N, K // 8), dtype=np.uint64).astype(np.uint32).view(np.int32)
    s = rng.integers(115, 125, size=(E, N, K // 32)).astype(np.uint8)
    ids = np.minimum(rng.zipf(1.3, size=rows) - 1, E + 1).astype(np.int32)
    rng.shuffle(ids)
    x = activations(rng, rows, K, "bf16")
    wt, st = dev(w), dev(s)
    y = ops.gather_qmm(x.reshape(rows, 1, K), wt, st, None, rhs_indices=dev(ids), group_size=32, bits=4, mode="mxfp4")
    used = np.unique(ids[ids < E])
    wv = {int(e): _mx.values(w[e], s[e], 4) for e in used}
    for e in np.unique(ids):
        at = np.flatnonzero(ids == e)
        rows_e = y[torch.from_numpy(at).cuda(), 0]
        if e >= E:
            assert (rows_e == 0).all()
        else:
            check_product(rows_e, host(x)[at], wv[int(e)], False, f"expert {e}")
    assert ops.device_error() == 0


@pytest.mark.parametrize("M", [1, 2, 3, 8, 12, 32])
@pytest.mark.parametrize("N,K", [(40000, 256), (30000, 544)])
def test_wide_products(ops, M, N, K):
    """Many tiles to a block, K within one ring of k-blocks and past a whole number of them."""
    rng = np.random.default_rng(M + K)
    w, s, wv = _mx.random_weights(rng, (N, K))
    x = activations(rng, M, K, "bf16")
    y = ops.quantized_matmul(x, dev(w), dev(s), None, group_size=32, bits=4, mode="mxfp4")
    check_product(y, host(x), wv, False)
    assert ops.device_error() == 0


def test_gather_promise_broken_is_contained(ops):
    """Ids that are not ascending after all: wrong rows, but nothing out of range, and later calls are right."""
    rng = np.random.default_rng(10)
    w, s, wv = _mx.random_weights(rng, (16, 128, 128))
    ids = rng.integers(-3, 20, size=200).astype(np.int32)
    x = activations(rng, 200, 128, "bf16")
    kw = dict(rhs_indices=dev(ids), group_size=32, bits=4, mode="mxfp4")
    ops.gather_qmm(x.reshape(200, 1, 128), dev(w), dev(s), None, sorted_indices=True, **kw)
    y = ops.gather_qmm(x.reshape(200, 1, 128), dev(w), dev(s), None, **kw)
    check_grouped(y, host(x), ids, np.arange(200), wv, False)


# --------------------------------------------------------------------------
# refusals
# --------------------------------------------------------------------------

def test_refusals(ops):
    x = torch.randn(4, 256, device="cuda", dtype=torch.bfloat16)
    w, s = ops.quantize(torch.randn(64, 256, device="cuda"), 32, 4, mode="mxfp4")
    xq, xs = ops.quantize(x, 32, 8, mode="mxfp8")
    kw = dict(group_size=32, bits=4, mode="mxfp4")
    for bad in (dict(kw, group_size=64), dict(kw, bits=8), dict(kw, mode="nvfp4"), dict(kw, transpose=False),
                dict(kw, mode="mxfp8", bits=8)):
        with pytest.raises(NotImplementedError):
            ops.quantized_matmul(x, w, s, None, **bad)
    with pytest.raises(NotImplementedError):
        ops.quantized_matmul(x.float(), w, s, None, **kw)
    for args in ((x, w, s, s), (x[:, :128], w, s, None), (x.cpu(), w, s, None), (x, w, s[:, :4], None),
                 (x, w, s.int(), None), (x, w.float(), s, None), (x, w[0], s, None)):
        with pytest.raises(ValueError):
            ops.quantized_matmul(*args, **kw)
    with pytest.raises(ValueError):
        ops.quantized_matmul(x, w, s, None, out=torch.empty(4, 63, device="cuda", dtype=x.dtype), **kw)
    with pytest.raises(ValueError):
        ops.mx_matmul(xq, xs[:, :4], w, s)
    with pytest.raises(NotImplementedError):
        ops.mx_matmul(xq, xs, w, s, dtype=torch.float32)
    with pytest.raises(ValueError):
        ops.mx_matmul(xq, xs, w, s, lhs_indices=torch.zeros(4, dtype=torch.int32, device="cuda"))
    bank, bs = w.reshape(2, 32, 32), s.reshape(2, 32, 8)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ops.gather_qmm(x.reshape(4, 1, 256), w, s, None, rhs_indices=ids, **kw)
    with pytest.raises(ValueError):
        ops.gather_qmm(x[:3].reshape(3, 1, 256), bank, bs, None, rhs_indices=ids, **kw)
    with pytest.raises(ValueError):
        ops.mx_matmul(xq[:3], xs[:3], bank, bs, rhs_indices=ids)  # fewer rows than ids, and no lhs_indices
    with pytest.raises(NotImplementedError):
        ops.mx_matmul(xq, xs, bank, bs, rhs_indices=ids, out=torch.empty(4, 32, device="cuda", dtype=x.dtype))
    for bad in (torch.randn(4, 48, device="cuda"), torch.randn(4, 64)):
        with pytest.raises(ValueError):
            ops.quantize(bad, 32, 4, mode="mxfp4")
    with pytest.raises(NotImplementedError):
        ops.quantize(torch.zeros(4, 64, device="cuda", dtype=torch.float64), 32, 4, mode="mxfp4")
    with pytest.raises(NotImplementedError):
        ops.quantize(x, 64, 4, mode="mxfp4")
    with pytest.raises(ValueError):
        ops.quantize(x, 32, 4, mode="mxfp4", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.dequantize(w, s, s, 32, 4, mode="mxfp4")
    with pytest.raises(ValueError):
        ops.dequantize(w, s[:, :3], None, 32, 4, mode="mxfp4")
    g = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    for args, extra in (((x, g[:128]), {}), ((x, g.half()), {}), ((x, g), {"residual": x[:2]}),
                        ((x, g), {"residual": x.half()}), ((x, g, -1.0), {}), ((x.cpu(), g), {})):
        with pytest.raises(ValueError):
            ops.rms_norm_quantize(*args, **extra)
    with pytest.raises(NotImplementedError):
        ops.rms_norm_quantize(x.float(), g.float())
