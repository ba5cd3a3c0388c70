"""The microscaled (MX) operators as workloads: what is timed, on which sizes, and their plain forms.

Five operators around weights and activations held as 4- and 8-bit floating-point codes with one
power-of-two scale per 32 values along the last axis:

  quantize   ops.quantize / ops.dequantize, mode "mxfp4" or "mxfp8": there and back
  norm       ops.rms_norm_quantize: residual addition, root-mean-square norm, mxfp8 rows
  matmul     ops.quantized_matmul, mode "mxfp4": bf16/fp16 activations times mxfp4 weights
  mx_matmul  ops.mx_matmul: mxfp8 activations times mxfp4 weights
  gather     ops.gather_qmm, mode "mxfp4": products grouped by expert, ragged group sizes

Format.  A block of 32 values v has amax = max|v| and the scale 2^e, e = floor(log2 amax) - emax
(emax 2 for the 4-bit type e2m1, 8 for the 8-bit type e4m3), clamped to [-127, 127] and stored as
the byte e + 127; a code is v * 2^-e rounded to nearest even and saturated at 6 or 448.  Codes are
packed low bits first into 32-bit words.

With ``own`` false, ``run`` computes the plain form in elementary torch operations in 32 bits; with
``own`` true it calls the package.  ``exact`` computes the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6


def listed():
    return [
        # activations of a verify batch to 8 bits (an odd number of rows)
        {"name": "quantize_act", "op": "quantize", "rows": 333, "k": 5120, "bits": 8, "dtype": "bf16"},
        # conversion of a decoder layer's largest projection to 4 bits
        {"name": "quantize_weight", "op": "quantize", "rows": 17408, "k": 5120, "bits": 4, "dtype": "bf16"},
        # the norm before a projection of a decoder layer, one token decoded
        {"name": "norm_decode", "op": "norm", "rows": 1, "k": 5120, "dtype": "bf16", "residual": True},
        # the same norm over a prefill chunk
        {"name": "norm_prefill", "op": "norm", "rows": 8192, "k": 5120, "dtype": "bf16", "residual": True},
        # one token through the smallest projection of a decoder layer (key / value heads): latency counts
        {"name": "matmul_decode", "op": "matmul", "m": 1, "n": 1024, "k": 5120, "dtype": "bf16"},
        # a speculative verify window through the largest projection
        {"name": "matmul_verify", "op": "matmul", "m": 5, "n": 17408, "k": 5120, "dtype": "f16"},
        # a long prefill chunk through the same projection
        {"name": "matmul_prefill", "op": "matmul", "m": 8192, "n": 17408, "k": 5120, "dtype": "bf16"},
        # a batch of sixteen decoded tokens through the down projection, activations in 8 bits
        {"name": "mx_matmul_decode", "op": "mx_matmul", "m": 16, "n": 5120, "k": 17408, "dtype": "bf16"},
        # a ragged prefill batch, activations in 8 bits
        {"name": "mx_matmul_prefill", "op": "mx_matmul", "m": 2011, "n": 17408, "k": 5120, "dtype": "bf16"},
        # one token's ten experts, gate and up projections in one bank
        {"name": "gather_decode", "op": "gather", "tokens": 1, "top_k": 10, "experts": 512, "n": 1024, "k": 2048,
         "dtype": "bf16", "skew": 0.0, "sorted": False},
        # a batch of decoded tokens through the down projections, ids in token order
        {"name": "gather_batch", "op": "gather", "tokens": 64, "top_k": 10, "experts": 512, "n": 2048, "k": 512,
         "dtype": "bf16", "skew": 1.0, "sorted": False},
        # a prefill chunk, rows sorted by expert, some experts with few rows and some with many
        {"name": "gather_prefill", "op": "gather", "tokens": 8192, "top_k": 10, "experts": 512, "n": 1024, "k": 2048,
         "dtype": "bf16", "skew": 1.0, "sorted": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "matmul", "mx_matmul", "gather"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 17408), "k": 32 * _log(rng, 2, 160), "bits": rng.choice([4, 8]),
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 8192), "k": 32 * _log(rng, 8, 160), "dtype": dtype,
                "residual": rng.random() < 0.75}
    if op in ("matmul", "mx_matmul"):
        n = _log(rng, 100, 17408)
        # most widths are whole numbers of 128; some only of 32
        k = 128 * _log(rng, 2, 136) if rng.random() < 0.8 else 32 * _log(rng, 5, 160)
        most = 8192 * 17408 * 5120
        return {"op": op, "m": min(_log(rng, 1, 8192), max(1, most // (n * k))), "n": n, "k": k, "dtype": dtype}
    experts = rng.choice([8, 32, 128, 256, 512])
    return {"op": op, "tokens": _log(rng, 1, 4096), "top_k": rng.randint(1, min(10, experts)), "experts": experts,
            "n": 8 * _log(rng, 16, 256), "k": 128 * _log(rng, 2, 16), "dtype": dtype,
            "skew": rng.choice([0.0, 1.0]), "sorted": rng.random() < 0.5}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _pow2(scales):
    """2^(byte - 127) in 32 bits, exact down to 2^-127."""
    byte = scales.to(torch.int32)
    return torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)


def _block_exponent(v, emax):
    """The stored scale byte of each block of 32 along the last axis of v (fp32), as int32."""
    amax = v.abs().amax(-1)
    return ((amax.view(torch.int32) >> 23) - emax).clamp_min(0)


def _encode(v, bits):
    """(codes uint8 [..., K], scale bytes uint8 [..., K/32]) of fp32 values."""
    b = v.reshape(*v.shape[:-1], -1, 32)
    byte = _block_exponent(b, 2 if bits == 4 else 8)
    a = torch.ldexp(b, (127 - byte).unsqueeze(-1))
    if bits == 8:
        code = a.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        m = a.abs()
        code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5)
                + (m > 5)) | (torch.signbit(a).to(torch.uint8) << 3)
    return code.reshape(v.shape), byte.to(torch.uint8)


def _pack(codes, bits):
    if bits == 4:
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return codes.contiguous().view(torch.int32)


def _quantized(gen, shape, bits, std):
    """Words and scales of normal values, drawn in parts so that the largest bank stays small in memory."""
    words, scales = [], []
    rows = shape[0]
    step = max(1, min(rows, (1 << 27) // max(1, math.prod(shape[1:]))))
    for r in range(0, rows, step):
        v = torch.randn((min(step, rows - r), *shape[1:]), generator=gen, device="cuda") * std
        c, s = _encode(v, bits)
        words.append(_pack(c, bits))
        scales.append(s)
    return torch.cat(words), torch.cat(scales)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    op = case["op"]
    s = {"case": case, "dtype": dt}
    if op == "quantize":
        std = 0.02 if case["bits"] == 4 else 1.0
        s["x"] = (torch.randn((case["rows"], case["k"]), generator=gen, device="cuda") * std).to(dt)
    elif op == "norm":
        shape = (case["rows"], case["k"])
        s["x"] = torch.randn(shape, generator=gen, device="cuda").to(dt)
        s["residual"] = (torch.randn(shape, generator=gen, device="cuda") * 4).to(dt) if case["residual"] else None
        s["weight"] = (1 + 0.1 * torch.randn(case["k"], generator=gen, device="cuda")).to(dt)
    elif op == "gather":
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        s["x"] = torch.randn((T, 1, case["k"]), generator=gen, device="cuda").to(dt)
        s["w"], s["scales"] = _quantized(gen, (E, case["n"], case["k"]), 4, 0.02)
        # a router's top-k: noise per token over a preference per expert
        pref = torch.randn((1, E), generator=gen, device="cuda") * case["skew"]
        noise = -torch.log(-torch.log(torch.rand((T, E), generator=gen, device="cuda").clamp(1e-6, 1 - 1e-6)))
        ids = (pref + noise).topk(k, dim=-1).indices.reshape(-1).to(torch.int32)
        src = torch.arange(T, device="cuda", dtype=torch.int32).repeat_interleave(k)
        if case["sorted"]:
            order = torch.argsort(ids, stable=True)
            ids, src = ids[order].contiguous(), src[order].contiguous()
        s["ids"], s["src"] = ids, src
    else:
        s["w"], s["scales"] = _quantized(gen, (case["n"], case["k"]), 4, 0.02)
        if op == "matmul":
            s["x"] = torch.randn((case["m"], case["k"]), generator=gen, device="cuda").to(dt)
        else:
            s["xq"], s["x_scales"] = _quantized(gen, (case["m"], case["k"]), 8, 1.0)
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _values4(words, scales):
    """fp32 values of packed mxfp4 words [..., K/8]."""
    byte = words.contiguous().view(torch.uint8)
    code = torch.stack([byte & 15, byte >> 4], -1).reshape(*scales.shape, 32)
    lut = torch.tensor(_E2M1, device=words.device)
    return (lut[code.to(torch.int32)] * _pow2(scales).unsqueeze(-1)).reshape(*words.shape[:-1], -1)


def _values8(words, scales):
    code = words.contiguous().view(torch.float8_e4m3fn).to(torch.float32)
    return (code.reshape(*scales.shape, 32) * _pow2(scales).unsqueeze(-1)).reshape(code.shape)


def _round_mx(v, bits):
    """fp32 values rounded to the blocks' 4- or 8-bit grid."""
    b = v.reshape(*v.shape[:-1], -1, 32)
    byte = _block_exponent(b, 2 if bits == 4 else 8)
    a = torch.ldexp(b, (127 - byte).unsqueeze(-1))
    if bits == 8:
        q = a.clamp(-448, 448).to(torch.float8_e4m3fn).to(torch.float32)
    else:
        # spacing 0.5 below 2, 1 up to 4, 2 up to 6; torch.round is to nearest even
        m = a.abs().clamp_max(6)
        step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
        q = torch.round(m / step) * step * torch.sign(a)
    return torch.ldexp(q, (byte - 127).unsqueeze(-1)).reshape(v.shape)


def _plain(s):
    case, dt, op = s["case"], s["dtype"], s["case"]["op"]
    if op == "quantize":
        return {"values": _round_mx(s["x"].float(), case["bits"]).to(dt)}
    if op == "norm":
        h = s["x"].float()
        if s["residual"] is not None:
            h = h + s["residual"].float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS) * s["weight"].float()
        out = {"values": _round_mx(y, 8).to(dt)}
        if s["residual"] is not None:
            out["h"] = h.to(dt)
        return out
    if op == "matmul":
        return {"y": (s["x"].float() @ _values4(s["w"], s["scales"]).T).to(dt)}
    if op == "mx_matmul":
        return {"y": (_values8(s["xq"], s["x_scales"]) @ _values4(s["w"], s["scales"]).T).to(dt)}
    # grouped: only the experts that have rows, each group padded to the largest
    used, group = torch.unique(s["ids"], return_inverse=True)
    order = torch.argsort(group, stable=True)
    counts = torch.bincount(group)
    first = torch.cumsum(counts, 0) - counts
    at = torch.empty_like(order)
    at[order] = torch.arange(order.numel(), device=order.device) - first[group[order]]
    x = torch.zeros((used.numel(), int(counts.max()), case["k"]), device=order.device)
    x[group, at] = s["x"][s["src"].long(), 0].float()
    y = x @ _values4(s["w"][used.long()], s["scales"][used.long()]).transpose(1, 2)
    return {"y": y[group, at].unsqueeze(1).to(dt)}


def _own(s):
    from mlxturbo_b200 import ops

    case, dt, op = s["case"], s["dtype"], s["case"]["op"]
    if op == "quantize":
        mode = "mxfp4" if case["bits"] == 4 else "mxfp8"
        wq, sc = ops.quantize(s["x"], 32, case["bits"], mode=mode)
        return {"values": ops.dequantize(wq, sc, None, 32, case["bits"], mode=mode, dtype=dt)}
    if op == "norm":
        xq, sc, h = ops.rms_norm_quantize(s["x"], s["weight"], _EPS, residual=s["residual"])
        out = {"values": ops.dequantize(xq, sc, None, 32, 8, mode="mxfp8", dtype=dt)}
        if h is not None:
            out["h"] = h
        return out
    if op == "matmul":
        return {"y": ops.quantized_matmul(s["x"], s["w"], s["scales"], None, group_size=32, bits=4, mode="mxfp4")}
    if op == "mx_matmul":
        return {"y": ops.mx_matmul(s["xq"], s["x_scales"], s["w"], s["scales"], dtype=dt)}
    return {"y": ops.gather_qmm(s["x"], s["w"], s["scales"], None, lhs_indices=s["src"], rhs_indices=s["ids"],
                                group_size=32, bits=4, mode="mxfp4", sorted_indices=case["sorted"])}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op == "quantize":  # values in, rounded values out
        n = case["rows"] * case["k"]
        return {"bytes": 2 * size * n, "flops": 3 * n}
    if op == "norm":  # row and residual in, new residual and normalised values out
        n = case["rows"] * case["k"]
        return {"bytes": (4 if case["residual"] else 2) * size * n + size * case["k"], "flops": 7 * n}
    n, k = case["n"], case["k"]
    weight = n * k * 17 // 32  # half a byte a value, one scale byte for 32
    if op == "gather":
        T, E, top = case["tokens"], case["experts"], case["top_k"]
        rows = T * top
        touched = min(E, rows, E * (1 - (1 - top / E) ** T) + 1e-9)  # experts met by evenly spread routing
        return {"bytes": touched * weight + T * k * 2 + rows * n * 2 + rows * 8, "flops": 2 * rows * n * k}
    m = case["m"]
    act = m * k * 2 if op == "matmul" else m * k * 33 // 32
    return {"bytes": weight + act + m * n * 2, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------

def _grid64(v, bits):
    """float64 values to the nearest point of their block's grid, ties to the even code."""
    emax, emin, mant, top = (2, 0, 1, 6.0) if bits == 4 else (8, -6, 3, 448.0)
    b = v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax).exponent - 1 - emax  # floor(log2 amax) - emax
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
    a = torch.ldexp(b, -e)
    p = (torch.frexp(a).exponent - 1).clamp_min(emin) - mant  # exponent of the grid's spacing around a
    q = torch.ldexp(torch.round(torch.ldexp(a, -p)), p).clamp(-top, top)
    return torch.ldexp(q, e).reshape(v.shape)


def _unpack64(words, scales, bits):
    """float64 values of packed words, field by field."""
    shift = torch.arange(0, 32, bits, device=words.device, dtype=torch.int32)
    code = (words.unsqueeze(-1) >> shift) & ((1 << bits) - 1)
    mant, bias = (1, 1) if bits == 4 else (3, 7)
    sign = 1.0 - 2.0 * (code >> (bits - 1)).double()
    field = (code >> mant) & ((1 << (bits - 1 - mant)) - 1)
    frac = (code & ((1 << mant) - 1)).double() / (1 << mant)
    frac = torch.where(field > 0, 1.0 + frac, 2.0 * frac)
    v = sign * torch.ldexp(frac, field - bias)
    v = v.reshape(*scales.shape, 32)
    return torch.ldexp(v, scales.to(torch.int32).unsqueeze(-1) - 127).reshape(*words.shape[:-1], -1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return {"values": _grid64(s["x"].double(), case["bits"])}
    if op == "norm":
        h = s["x"].double() + (s["residual"].double() if s["residual"] is not None else 0.0)
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + _EPS) * s["weight"].double()
        out = {"values": _grid64(y, 8)}
        if s["residual"] is not None:
            out["h"] = h
        return out
    if op == "matmul":
        return {"y": s["x"].double() @ _unpack64(s["w"], s["scales"], 4).T}
    if op == "mx_matmul":
        return {"y": _unpack64(s["xq"], s["x_scales"], 8) @ _unpack64(s["w"], s["scales"], 4).T}
    y = torch.empty((s["ids"].numel(), 1, case["n"]), dtype=torch.float64, device="cuda")
    for e in torch.unique(s["ids"]).tolist():
        at = (s["ids"] == e).nonzero().reshape(-1)
        y[at, 0] = s["x"][s["src"][at].long(), 0].double() @ _unpack64(s["w"][e], s["scales"][e], 4).T
    return {"y": y}
