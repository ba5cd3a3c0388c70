"""The microscaled formats through the modules, the dispatcher, a checkpoint and the example layer."""

import json
import os
import sys

import numpy as np
import pytest
import torch

import _mx

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MX = dict(group_size=32, bits=4, mode="mxfp4")


def test_layers_hold_mxfp4_weights_on_the_host():
    """Shapes, types and refusals need no GPU."""
    from mlxturbo_b200 import nn

    layer = nn.QuantizedLinear(256, 64, True, **MX)
    assert layer.weight.shape == (64, 32) and layer.scales.shape == (64, 8) and layer.scales.dtype == torch.uint8
    assert layer.biases is None and layer.bias.dtype == torch.bfloat16
    assert set(layer.state_dict()) == {"weight", "scales", "bias"}
    glu = nn.SwitchGLU(256, 64, 4, **MX)
    assert glu.down_proj.weight.shape == (4, 256, 8) and glu.slice_experts(1, 3).up_proj.num_experts == 2
    with pytest.raises(NotImplementedError):
        glu.fused_gate_up()
    for bad in (dict(MX, group_size=64), dict(MX, bits=8), dict(MX, mode="nvfp4")):
        with pytest.raises(NotImplementedError):
            nn.QuantizedLinear(256, 64, **bad)
    with pytest.raises(NotImplementedError):
        nn.QuantizedLinear(256, 64).forward_mx(None, None)


def test_checkpoint_with_mxfp4_layers(tmp_path):
    from mlxturbo_b200 import checkpoint as ck

    rng = np.random.default_rng(0)
    w, s, _ = _mx.random_weights(rng, (64, 128))
    bw, bs, _ = _mx.random_weights(rng, (3, 32, 128))
    ck.write_safetensors(str(tmp_path / "model.safetensors"), {
        "a.weight": torch.from_numpy(w), "a.scales": torch.from_numpy(s),
        "b.weight": torch.from_numpy(bw), "b.scales": torch.from_numpy(bs),
        "c.weight": torch.zeros(8, 16, dtype=torch.int32), "c.scales": torch.ones(8, 2, dtype=torch.bfloat16),
        "c.biases": torch.zeros(8, 2, dtype=torch.bfloat16)})
    (tmp_path / "config.json").write_text(json.dumps({"quantization": {
        "group_size": 32, "bits": 4, "mode": "mxfp4", "c": {"group_size": 64, "bits": 4, "mode": "affine"}}}))
    layers, _ = ck.load_model_dir(str(tmp_path))
    assert layers["a"].mode == "mxfp4" and torch.equal(layers["a"].scales, torch.from_numpy(s))
    assert layers["b"].weight.shape == (3, 32, 16) and layers["b"].biases is None
    assert layers["c"].mode == "affine" and layers["c"].biases is not None
    with pytest.raises(ValueError):
        ck.load_quantized_linear({"a.weight": torch.from_numpy(w), "a.scales": torch.from_numpy(s)}, "a", 32, 4)


@pytest.mark.gpu
def test_linear_and_switch_layers():
    from mlxturbo_b200 import nn, ops
    from mlxturbo_b200.kernels import dispatch

    torch.manual_seed(1)
    w = torch.randn(192, 256, device="cuda") * 0.05
    bias = torch.randn(192, device="cuda")
    layer = nn.QuantizedLinear.from_float(w, bias, **MX)
    x = torch.randn(7, 256, device="cuda", dtype=torch.bfloat16)
    want = ops.quantized_matmul(x, layer.weight, layer.scales, None, **MX) + layer.bias
    assert torch.equal(layer(x), want)
    model = torch.nn.Sequential(layer)
    dispatch.enable(model)
    assert torch.equal(model(x), want)
    xq, xs = ops.quantize(x, 32, 8, mode="mxfp8")
    back = ops.dequantize(xq, xs, None, 32, 8, mode="mxfp8")
    assert torch.allclose(layer.forward_mx(xq, xs).float(), layer(back).float(), rtol=2.0 ** -7, atol=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_moe_block(tokens):
    """moe_combine_fold over mxfp4 experts against the experts one by one in fp32."""
    from mlxturbo_b200 import moe, nn, ops

    torch.manual_seed(tokens)
    E, H, I, top = 8, 256, 128, 2
    glu = nn.SwitchGLU(H, I, E, device="cuda", **MX)
    deq = {}
    for name in ("gate_proj", "up_proj", "down_proj"):
        bank = getattr(glu, name)
        n, k = bank.weight.shape[1], bank.weight.shape[2] * 8
        wq, s = ops.quantize(torch.randn(E, n, k, device="cuda") * 0.05, 32, 4, mode="mxfp4")
        bank.weight.copy_(wq)
        bank.scales.copy_(s)
        deq[name] = ops.dequantize(wq, s, None, 32, 4, mode="mxfp4", dtype=torch.float32)
    x = torch.randn(tokens, H, device="cuda", dtype=torch.bfloat16)
    ids = torch.stack([torch.randperm(E, device="cuda")[:top] for _ in range(tokens)]).to(torch.int32)
    wts = torch.rand(tokens, top, device="cuda")
    y = moe.moe_combine_fold(glu, x, ids, wts)
    want = torch.zeros(tokens, H, device="cuda")
    for t in range(tokens):
        for k in range(top):
            e = int(ids[t, k])
            a = torch.nn.functional.silu(deq["gate_proj"][e] @ x[t].float()) * (deq["up_proj"][e] @ x[t].float())
            want[t] += wts[t, k] * (deq["down_proj"][e] @ a)
    # roundings to bf16 (2^-9 each) of gate, up, their product, the weighted product, the result of down
    # and the sum: well under 2^-5 of the values' size
    assert (y.float() - want).abs().max() <= 2.0 ** -5 * want.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 24, 300])
def test_example_layer(tokens):
    sys.path.insert(0, os.path.join(REPO, "examples"))
    import mxfp4_layer as ex

    torch.manual_seed(tokens)
    layer = ex.Layer(512, 768, 16, 256, 4)
    x = torch.randn(tokens, 512, device="cuda", dtype=torch.bfloat16)
    r = torch.randn(tokens, 512, device="cuda", dtype=torch.bfloat16)
    y, h = layer(x, r)
    y_ref, h_ref = layer.reference(x, r)
    # bf16 roundings (2^-9) of a few intermediates; a value between two 8-bit codes may take the other one
    # (2^-4 of it, in few places), and a token may take another last expert when two are as likely
    assert (h.float() - h_ref).norm() <= 2.0 ** -6 * h_ref.norm()
    row = (y.float() - y_ref).norm(dim=-1) / y_ref.norm(dim=-1)
    assert row.median() <= 2.0 ** -4 and (row > 2.0 ** -3).float().mean() <= 0.05
