"""The type of a quantized layer's activations follows the module (no GPU)."""

import copy

import pytest
import torch

from mlxturbo_b200 import nn

MX = dict(group_size=32, bits=4, mode="mxfp4")


@pytest.mark.parametrize("kw", [{}, MX])
def test_experts_sliced_from_a_converted_bank(kw):
    """A bank converted to fp16 gives fp16 slices with the same scales, biases and bias."""
    bank = nn.QuantizedSwitchLinear(128, 32, 4, True, **kw)
    bank = bank.half()
    if not kw:
        bank.scales.copy_(torch.rand(bank.scales.shape))
        bank.biases.copy_(torch.rand(bank.biases.shape))
    bank.bias.data.copy_(torch.rand(bank.bias.shape))
    part = bank.slice_experts(1, 3)
    assert part.dtype == part.bias.dtype == torch.float16 and torch.equal(part.bias, bank.bias[1:3])
    assert part.scales.dtype == bank.scales.dtype and torch.equal(part.scales, bank.scales[1:3])
    if not kw:
        assert part.biases.dtype == torch.float16 and torch.equal(part.biases, bank.biases[1:3])


@pytest.mark.parametrize("make", [lambda **kw: nn.QuantizedLinear(64, 32, True, **kw),
                                  lambda **kw: nn.QuantizedSwitchLinear(64, 32, 3, True, **kw)])
@pytest.mark.parametrize("kw", [{}, MX])
def test_dtype_follows_conversions(make, kw):
    layer = make(**kw)
    assert layer.dtype == torch.bfloat16
    names = set(layer.state_dict())
    layer.half()
    assert layer.dtype == layer.bias.dtype == torch.float16
    assert copy.deepcopy(layer).dtype == torch.float16
    layer.to(torch.bfloat16)
    assert layer.dtype == layer.bias.dtype == torch.bfloat16
    assert set(layer.state_dict()) == names == {"weight", "scales", "bias"} | ({"biases"} if not kw else set())
    assert layer.weight.dtype == torch.int32 and (not kw or layer.scales.dtype == torch.uint8)
    assert make(**kw, dtype=torch.float16).dtype == torch.float16
