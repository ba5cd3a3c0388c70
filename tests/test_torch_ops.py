"""How the operators stand in PyTorch's dispatcher: one kernel per device, below autograd and the dispatch modes."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from mlxturbo_b200 import _lib

NAMES = ["quantized_matmul", "quantized_matmul_out", "mx_quantize", "mx_dequantize", "mx_rms_norm", "mx_matmul",
         "mx_matmul_out", "mx_gather"]


@pytest.mark.parametrize("name", NAMES)
def test_registered_per_device(name):
    assert _lib.torch_ops() is not None
    has = lambda key: torch._C._dispatch_has_kernel_for_dispatch_key(f"mlxturbo_b200::{name}", key)  # noqa: E731
    assert has("CUDA") and has("CPU") and not has("CompositeImplicitAutograd")


def test_all_cpu_arguments_are_refused():
    from mlxturbo_b200 import ops

    x, g = torch.randn(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    w, s = torch.zeros(8, 8, dtype=torch.int32), torch.zeros(8, 2, dtype=torch.uint8)
    xq, xs = torch.zeros(4, 16, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.uint8)
    ids = torch.zeros(4, dtype=torch.int32)
    kw = dict(group_size=32, bits=4, mode="mxfp4")
    calls = [lambda: ops.quantize(x, **kw), lambda: ops.dequantize(w, s, None, **kw),
             lambda: ops.rms_norm_quantize(x, g), lambda: ops.rms_norm_quantize(x, g, residual=x),
             lambda: ops.quantized_matmul(x, w, s, None, **kw),
             lambda: ops.quantized_matmul(x, w, s, None, out=torch.empty(4, 8, dtype=torch.bfloat16), **kw),
             lambda: ops.mx_matmul(xq, xs, w, s),
             lambda: ops.mx_matmul(xq, xs, w[None], s[None], rhs_indices=ids),
             lambda: ops.gather_qmm(x[:, None], w[None], s[None], None, rhs_indices=ids, **kw)]
    for call in calls:
        with pytest.raises(ValueError):
            call()


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func._schema.name)
        return func(*args, **(kwargs or {}))


@pytest.mark.gpu
def test_autograd_and_modes_see_the_calls():
    """A gradient through an MX operator is refused aloud, as through the affine one, and a mode is asked."""
    from mlxturbo_b200 import ops

    x = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16)
    g = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    w, s = ops.quantize(torch.randn(8, 64, device="cuda"), 32, 4, mode="mxfp4")
    aw, asc, ab = ops.quantize(torch.randn(8, 64, device="cuda"), 64, 4, dtype=torch.bfloat16)
    kw = dict(group_size=32, bits=4, mode="mxfp4")
    xg = x.clone().requires_grad_()
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    affine = ops.quantized_matmul(xg, aw, asc, ab)
    results = [(ops.quantized_matmul(xg, w, s, None, **kw), ops.quantized_matmul(x, w, s, None, **kw)),
               (ops.gather_qmm(xg[:, None], w[None], s[None], None, rhs_indices=ids, **kw),
                ops.gather_qmm(x[:, None], w[None], s[None], None, rhs_indices=ids, **kw)),
               (ops.rms_norm_quantize(xg, g, residual=x)[2], ops.rms_norm_quantize(x, g, residual=x)[2])]
    for y, plain in results:
        assert torch.equal(y, plain)
        assert y.requires_grad == affine.requires_grad
        assert type(y.grad_fn) is type(affine.grad_fn)
    xq, xs, h = ops.rms_norm_quantize(xg, g)  # no residual: no sum to give back
    assert h is None and torch.equal(xq, ops.rms_norm_quantize(x, g)[0])
    with Seen() as seen:
        ops.quantized_matmul(x, w, s, None, **kw)
        ops.rms_norm_quantize(x, g)
    assert seen.names == ["mlxturbo_b200::mx_matmul", "mlxturbo_b200::mx_rms_norm"]


@pytest.mark.gpu
def test_operators_under_inference_and_no_grad():
    from mlxturbo_b200 import ops

    x = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16)
    w, s = ops.quantize(torch.randn(8, 64, device="cuda"), 32, 4, mode="mxfp4")
    want = ops.quantized_matmul(x, w, s, None, group_size=32, bits=4, mode="mxfp4")
    for context in (torch.no_grad, torch.inference_mode):
        with context():
            xg = x.clone().requires_grad_()
            y = ops.quantized_matmul(xg, w, s, None, group_size=32, bits=4, mode="mxfp4")
            assert torch.equal(y, want) and not y.requires_grad
