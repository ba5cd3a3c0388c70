"""MLX model directories that mix microscaled and affine layers (no GPU)."""

import json

import numpy as np
import pytest
import torch

import _mx
from mlxturbo_b200 import checkpoint as ck


def model_dir(path, quantization, tensors, **config):
    ck.write_safetensors(str(path / "model.safetensors"), tensors)
    (path / "config.json").write_text(json.dumps({"quantization": quantization, **config}))
    return str(path)


def mx_layer(name, n=64, k=128, seed=0):
    w, s, _ = _mx.random_weights(np.random.default_rng(seed), (n, k))
    return {f"{name}.weight": torch.from_numpy(w), f"{name}.scales": torch.from_numpy(s)}


def affine_layer(name, n=8, k=128, group=64, bits=8, dtype=torch.bfloat16):
    return {f"{name}.weight": torch.arange(n * k * bits // 32, dtype=torch.int32).reshape(n, -1),
            f"{name}.scales": torch.ones(n, k // group, dtype=dtype),
            f"{name}.biases": torch.zeros(n, k // group, dtype=dtype)}


MX = {"group_size": 32, "bits": 4, "mode": "mxfp4"}


def test_override_without_a_mode_is_affine(tmp_path):
    """Attention or a router in 8 bits beside mxfp4 experts, the override as MLX writes it."""
    t = {**mx_layer("a"), **affine_layer("attn")}
    layers, qc = ck.load_model_dir(model_dir(tmp_path, {**MX, "attn": {"group_size": 64, "bits": 8}}, t))
    assert layers["a"].mode == "mxfp4" and layers["attn"].mode == "affine"
    assert (layers["attn"].group_size, layers["attn"].bits) == (64, 8)
    assert torch.equal(layers["attn"].weight, t["attn.weight"]) and torch.equal(layers["attn"].scales, t["attn.scales"])
    assert qc.mode_for_layer("attn") == "affine" and qc.mode_for_layer("other") == "mxfp4"


def test_override_of_an_mxfp4_layer(tmp_path):
    """With its mode, in an affine model; without one but without biases too, in an mxfp4 model."""
    t = {**mx_layer("a"), **affine_layer("b", bits=4)}
    layers, _ = ck.load_model_dir(model_dir(tmp_path, {"group_size": 64, "bits": 4, "a": MX}, t))
    assert layers["a"].mode == "mxfp4" and layers["b"].mode == "affine"
    layers, _ = ck.load_model_dir(model_dir(tmp_path, {**MX, "a": {"group_size": 32, "bits": 4}, "b": {
        "group_size": 64, "bits": 4}}, t))
    assert layers["a"].mode == "mxfp4" and layers["b"].mode == "affine"


def test_mode_that_the_tensors_contradict(tmp_path):
    with pytest.raises(ValueError):
        ck.load_model_dir(model_dir(tmp_path, {"group_size": 32, "bits": 4}, mx_layer("a")))
    with pytest.raises(ValueError):
        ck.load_model_dir(model_dir(tmp_path, {**MX, "b": dict(MX)}, affine_layer("b", bits=4, group=32)))


@pytest.mark.parametrize("config", [{"torch_dtype": "float16"}, {"dtype": "float16"}, {}])
def test_layers_of_an_fp16_model(tmp_path, config):
    """mxfp4 tensors do not say the activations' type: the model does, or the bias, which keeps its bits."""
    bias = (torch.randn(64, generator=torch.Generator().manual_seed(1)) / 3).half()
    t = {**mx_layer("a"), "a.bias": bias, **mx_layer("b"), **affine_layer("c", dtype=torch.float16)}
    layers, _ = ck.load_model_dir(model_dir(tmp_path, {**MX, "c": {"group_size": 64, "bits": 8}}, t, **config))
    assert layers["a"].bias.dtype == torch.float16 and torch.equal(layers["a"].bias.data, bias)
    assert layers["a"].dtype == torch.float16 and layers["c"].scales.dtype == torch.float16
    assert layers["b"].dtype == (torch.float16 if config else torch.bfloat16)
    layers, _ = ck.load_model_dir(model_dir(tmp_path, {**MX, "c": {"group_size": 64, "bits": 8}}, t, **config),
                                  dtype=torch.bfloat16)
    assert layers["a"].dtype == layers["a"].bias.dtype == layers["b"].dtype == torch.bfloat16


def test_dtype_of_one_layer():
    t = {**mx_layer("a"), "a.bias": torch.zeros(64, dtype=torch.float16)}
    assert ck.load_quantized_linear(t, "a", 32, 4, mode="mxfp4").dtype == torch.float16
    assert ck.load_quantized_linear(t, "a", 32, 4, mode="mxfp4", dtype=torch.bfloat16).dtype == torch.bfloat16
    t["a.bias"] = t["a.bias"].float()
    assert ck.load_quantized_linear(t, "a", 32, 4, mode="mxfp4").dtype == torch.bfloat16
