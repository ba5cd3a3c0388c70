"""MLX quantized checkpoints (safetensors + config.json) loaded straight into
the quantized layers, with no repacking.

``mx.quantize`` / mlx-lm ``convert`` write every quantized linear as three
tensors, ``<prefix>.weight`` (U32 [N, K*bits/32]), ``<prefix>.scales`` and
``<prefix>.biases`` (the activation dtype, [N, K/group_size]); expert banks
carry a leading expert axis.  config.json's ``"quantization"`` holds the
default ``group_size`` / ``bits`` and optional per-layer overrides keyed by
the layer prefix (how the reference's re-quantiser writes mixed bit widths,
mlxturbo/rebit.py:96-124).  The kernels consume that layout as is, so a
checkpoint's bytes are the tensors the layers hold.

The safetensors container is read here directly: an 8-byte little-endian
header length, a JSON header of ``{name: {dtype, shape, data_offsets}}`` and
the raw little-endian data.
"""

from __future__ import annotations

import json
import os
import struct
from typing import Iterable

import numpy as np
import torch

from .nn import QuantizedLinear, QuantizedSwitchLinear

# safetensors dtype -> (numpy dtype of the raw bytes, torch dtype to present)
_DTYPES = {
    "U32": (np.int32, torch.int32),  # uint32 codes carried as int32 bit patterns (torch has no CUDA uint32 math)
    "I32": (np.int32, torch.int32),
    "BF16": (np.int16, torch.bfloat16),
    "F16": (np.float16, torch.float16),
    "F32": (np.float32, torch.float32),
    "I64": (np.int64, torch.int64),
    "U8": (np.uint8, torch.uint8),
    "I8": (np.int8, torch.int8),
    "BOOL": (np.bool_, torch.bool),
}
_TORCH_TO_ST = {torch.bfloat16: "BF16", torch.float16: "F16", torch.float32: "F32", torch.int32: "I32",
                torch.int64: "I64", torch.uint8: "U8", torch.int8: "I8", torch.bool: "BOOL"}

_HALF = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def read_header(path: str) -> tuple[dict, int]:
    """(header dict, byte offset of the data section)."""
    with open(path, "rb") as f:
        (n,) = struct.unpack("<Q", f.read(8))
        header = json.loads(f.read(n))
    return header, 8 + n


def read_safetensors(path: str, names: Iterable[str] | None = None, device=None) -> dict[str, torch.Tensor]:
    """Tensors of a .safetensors file (all, or `names`), on `device` (default CPU).

    U32 tensors come back as int32 tensors holding the same bits.
    """
    header, base = read_header(path)
    want = set(names) if names is not None else None
    mm = np.memmap(path, dtype=np.uint8, mode="r")
    out = {}
    for name, meta in header.items():
        if name == "__metadata__" or (want is not None and name not in want):
            continue
        try:
            np_dt, t_dt = _DTYPES[meta["dtype"]]
        except KeyError:
            raise NotImplementedError(f"{name}: safetensors dtype {meta['dtype']} is not supported") from None
        b0, b1 = meta["data_offsets"]
        raw = np.array(mm[base + b0:base + b1])  # copy out of the map
        arr = raw.view(np_dt).reshape(meta["shape"])
        t = torch.from_numpy(arr)
        if t_dt is torch.bfloat16:
            t = t.view(torch.bfloat16)
        out[name] = t if device is None else t.to(device)
    if want is not None and want - set(out):
        raise KeyError(f"{sorted(want - set(out))} not in {path}")
    return out


def write_safetensors(path: str, tensors: dict[str, torch.Tensor], metadata: dict[str, str] | None = None,
                      u32: Iterable[str] = ()) -> None:
    """Write tensors (CPU or CUDA) to a .safetensors file; names in `u32` are stored as U32."""
    u32 = set(u32)
    header: dict = {}
    blobs = []
    off = 0
    for name in sorted(tensors):
        t = tensors[name].detach().contiguous().cpu()
        if name in u32:
            if t.dtype not in (torch.int32, getattr(torch, "uint32", torch.int32)):
                raise ValueError(f"{name}: U32 needs 32-bit integer data")
            dt = "U32"
            data = t.view(torch.int32).numpy().tobytes()
        else:
            dt = _TORCH_TO_ST.get(t.dtype)
            if dt is None:
                raise NotImplementedError(f"{name}: dtype {t.dtype}")
            data = (t.view(torch.int16) if t.dtype is torch.bfloat16 else t).numpy().tobytes()
        header[name] = {"dtype": dt, "shape": list(t.shape), "data_offsets": [off, off + len(data)]}
        blobs.append(data)
        off += len(data)
    if metadata:
        header["__metadata__"] = dict(metadata)
    hb = json.dumps(header, separators=(",", ":")).encode()
    hb += b" " * (-len(hb) % 8)  # keep the data section 8-byte aligned
    with open(path, "wb") as f:
        f.write(struct.pack("<Q", len(hb)))
        f.write(hb)
        for b in blobs:
            f.write(b)


class QuantConfig:
    """config.json's "quantization": default group_size/bits plus per-prefix overrides.

    ``dtype``: the model's own ("torch_dtype" or "dtype") where it is a 16-bit one, else None."""

    def __init__(self, quantization: dict | None, dtype: torch.dtype | None = None):
        self.dtype = dtype
        q = dict(quantization or {})
        self.group_size = int(q.pop("group_size", 64))
        self.bits = int(q.pop("bits", 4))
        self.mode = q.pop("mode", "affine")
        self.overrides = {k: v for k, v in q.items() if isinstance(v, dict)}

    @classmethod
    def from_model_dir(cls, model_dir: str) -> "QuantConfig":
        with open(os.path.join(model_dir, "config.json")) as f:
            cfg = json.load(f)
        dtype = _HALF.get(str(cfg.get("torch_dtype") or cfg.get("dtype")))
        return cls(cfg.get("quantization") or cfg.get("quantization_config"), dtype)

    def for_layer(self, prefix: str) -> tuple[int, int]:
        o = self.overrides.get(prefix)
        if o is None:
            return self.group_size, self.bits
        return int(o.get("group_size", self.group_size)), int(o.get("bits", self.bits))

    def mode_for_layer(self, prefix: str, biases: bool = True) -> str:
        """The layer's mode; `biases`: whether the layer has such a tensor.

        An override stands for the whole of a layer's settings in MLX, whose mode
        defaults to affine whatever the model's.  A layer without biases cannot be
        affine and takes the model's.
        """
        o = self.overrides.get(prefix)
        if o is None or not (biases or "mode" in o):
            return self.mode
        return o.get("mode", "affine")


def quantized_prefixes(tensors: dict[str, torch.Tensor]) -> list[str]:
    """Prefixes that carry a (weight, scales, biases) triple, or (mxfp4) weight and scales."""
    return sorted(n[: -len(".scales")] for n in tensors
                  if n.endswith(".scales") and n[: -len(".scales")] + ".weight" in tensors)


def _check(prefix: str, w: torch.Tensor, s: torch.Tensor, b: torch.Tensor | None, group_size: int, bits: int,
           mode: str) -> int:
    K = w.shape[-1] * 32 // bits
    if (b is None) != (mode != "affine"):
        raise ValueError(f"{prefix}: mode {mode!r} {'needs' if b is None else 'has no'} biases")
    if w.shape[-1] * 32 != K * bits or K % group_size or s.shape[-1] != K // group_size or (
            b is not None and b.shape != s.shape):
        raise ValueError(f"{prefix}: weight {tuple(w.shape)} / scales {tuple(s.shape)} do not match "
                         f"bits={bits} group_size={group_size}")
    return K


def _layer_dtype(s: torch.Tensor, bias: torch.Tensor | None, mode: str, dtype: torch.dtype | None) -> torch.dtype:
    if mode == "affine":
        return s.dtype
    if dtype is None and bias is not None and bias.dtype in _HALF.values():
        return bias.dtype
    return dtype or torch.bfloat16


def load_quantized_linear(tensors: dict[str, torch.Tensor], prefix: str, group_size: int = 64, bits: int = 4,
                          device=None, mode: str = "affine", dtype: torch.dtype | None = None) -> QuantizedLinear:
    """A QuantizedLinear from `<prefix>.weight/.scales/.biases` (+ `.bias` if present).

    `dtype` is the activations' of an mxfp4 layer (default: the bias's if 16-bit, else
    bfloat16); an affine one's is its scales'."""
    w, s, b = tensors[f"{prefix}.weight"], tensors[f"{prefix}.scales"], tensors.get(f"{prefix}.biases")
    K = _check(prefix, w, s, b, group_size, bits, mode)
    dev = device if device is not None else w.device
    bias = tensors.get(f"{prefix}.bias")
    layer = QuantizedLinear(K, w.shape[0], bias is not None, group_size, bits, mode,
                            dtype=_layer_dtype(s, bias, mode, dtype), device=dev)
    layer.weight.copy_(w.view(torch.int32))
    layer.scales.copy_(s)
    if b is not None:
        layer.biases.copy_(b)
    if bias is not None:
        layer.bias.data.copy_(bias)
    return layer


def load_switch_linear(tensors: dict[str, torch.Tensor], prefix: str, group_size: int = 64, bits: int = 4,
                       device=None, mode: str = "affine", dtype: torch.dtype | None = None) -> QuantizedSwitchLinear:
    """A QuantizedSwitchLinear (expert bank, leading E axis) from its tensors."""
    w, s, b = tensors[f"{prefix}.weight"], tensors[f"{prefix}.scales"], tensors.get(f"{prefix}.biases")
    K = _check(prefix, w, s, b, group_size, bits, mode)
    dev = device if device is not None else w.device
    bias = tensors.get(f"{prefix}.bias")
    layer = QuantizedSwitchLinear(K, w.shape[1], w.shape[0], bias is not None, group_size, bits, mode,
                                  dtype=_layer_dtype(s, bias, mode, dtype), device=dev)
    layer.weight.copy_(w.view(torch.int32))
    layer.scales.copy_(s)
    if b is not None:
        layer.biases.copy_(b)
    if bias is not None:
        layer.bias.data.copy_(bias)
    return layer


def load_model_dir(model_dir: str, device=None,
                   dtype: torch.dtype | None = None) -> tuple[dict[str, torch.nn.Module], QuantConfig]:
    """Every quantized layer of an MLX model directory (*.safetensors + config.json).

    Returns {prefix: QuantizedLinear or QuantizedSwitchLinear} (a 3-D weight is
    an expert bank) and the quantization config.  `dtype` is the activations' of
    its mxfp4 layers (default: the model's, else the bias's if 16-bit, else
    bfloat16).
    """
    qc = QuantConfig.from_model_dir(model_dir)
    layers: dict[str, torch.nn.Module] = {}
    for fn in sorted(os.listdir(model_dir)):
        if not fn.endswith(".safetensors"):
            continue
        t = read_safetensors(os.path.join(model_dir, fn))
        for prefix in quantized_prefixes(t):
            gs, bits = qc.for_layer(prefix)
            load = load_switch_linear if t[f"{prefix}.weight"].dim() == 3 else load_quantized_linear
            layers[prefix] = load(t, prefix, gs, bits, device=device,
                                  mode=qc.mode_for_layer(prefix, f"{prefix}.biases" in t), dtype=dtype or qc.dtype)
    return layers, qc


__all__ = [
    "QuantConfig", "load_model_dir", "load_quantized_linear", "load_switch_linear", "quantized_prefixes",
    "read_header", "read_safetensors", "write_safetensors",
]
