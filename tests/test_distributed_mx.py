"""Sharded layers and microscaled weights (no GPU)."""

import pytest
import torch

from mlxturbo_b200 import distributed as D
from mlxturbo_b200 import nn

MX = dict(group_size=32, bits=4, mode="mxfp4")


@pytest.mark.parametrize("cls", [D.QuantizedAllToShardedLinear, D.QuantizedShardedToAllLinear, D.ColumnShardedLMHead])
def test_sharded_linears_refuse_mxfp4_weights(cls):
    layer = nn.QuantizedLinear(256, 64, **MX)
    with pytest.raises(NotImplementedError, match="affine"):
        cls.from_full(layer.weight, layer.scales, layer.biases, group_size=32, bits=4)
    with pytest.raises(NotImplementedError, match="affine"):
        cls(layer.weight, layer.scales, layer.biases, None, 32, 4, None, None)


def test_experts_are_split_with_mxfp4_weights():
    glu = nn.SwitchGLU(256, 64, 4, **MX)
    glu.up_proj.scales.copy_(torch.randint(0, 255, glu.up_proj.scales.shape))
    part = D.ExpertParallelSwitchGLU.from_full(glu)
    assert part.glu.up_proj.mode == "mxfp4" and torch.equal(part.glu.up_proj.scales, glu.up_proj.scales)
