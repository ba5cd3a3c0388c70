"""The microscaled formats and their products in 64 bits (CPU), for the tests.

Codes are looked up in tables written out from the formats' definition, and a
value is rounded by searching the table, so nothing here shares a method with
the kernels.
"""

from __future__ import annotations

import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
                 for e in range(16) for m in range(8)][:127])  # code 127 is NaN


def table(bits):
    t = E2M1 if bits == 4 else np.append(E4M3, np.nan)
    return np.concatenate([t, -t])


def quantize(v, bits):
    """(codes uint8 [.., K], scale bytes uint8 [.., K/32]) of float64 values."""
    v = np.asarray(v, np.float64)
    b = v.reshape(*v.shape[:-1], -1, 32)
    grid, emax = (E2M1, 2) if bits == 4 else (E4M3, 8)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    amax = np.abs(b).max(-1)
    e = np.where(amax > 0, np.frexp(amax)[1] - 1 - emax, -127).clip(-127, 127)
    a = np.abs(np.ldexp(b, -e[..., None]))
    mid = (grid[1:] + grid[:-1]) / 2
    # a tie goes to the even code: the upper one when the lower one is odd
    lo = np.searchsorted(mid, a, side="left")
    hi = np.searchsorted(mid, a, side="right")
    code = np.where((lo != hi) & (lo % 2 == 1), hi, lo)
    code = (code + np.where(np.signbit(b), 1 << (bits - 1), 0)).astype(np.uint8)
    code[bad] = 0
    scale = np.where(bad, 255, e + 127).astype(np.uint8)
    return code.reshape(v.shape), scale


def pack(code, bits):
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return np.ascontiguousarray(code).view("<u4").view(np.int32)


def values(words, scales, bits):
    """float64 values of packed words and scale bytes (torch or numpy)."""
    w = words.cpu().numpy() if isinstance(words, torch.Tensor) else words
    s = (scales.cpu().numpy() if isinstance(scales, torch.Tensor) else scales).astype(np.int64)
    byte = np.ascontiguousarray(w).view(np.uint8)
    code = np.stack([byte & 15, byte >> 4], -1).reshape(*byte.shape[:-1], -1) if bits == 4 else byte
    v = table(bits)[code].reshape(*s.shape, 32)
    v = np.ldexp(v, (s - 127)[..., None])
    v[s == 255] = np.nan
    return v.reshape(code.shape)


def random_weights(rng, shape, bits=4, std=0.02):
    """Packed words, scale bytes and the values they stand for."""
    code, scale = quantize(rng.normal(0, std, size=shape), bits)
    w = pack(code, bits)
    return w, scale, values(w, scale, bits)


def product_bound(x, w, ref, f16):
    """Largest |y - ref| of a product with fp32 sums, rounded once to 16 bits.

    x [M, K], w [N, K], ref = x @ w^T in 64 bits.  The rounding of the result
    costs half a unit in the last place.  The sum takes one fp32 addition for
    each 16 products at most often, each off by at most 2^-23 of the running
    sum, itself at most S = sum |x||w|; eight more for joining parts of the sum.
    Activations may be held to 2^-21 of the largest of their block of 32.
    """
    ax, aw = np.abs(x), np.abs(w)
    S = ax @ aw.T
    top = np.repeat(ax.reshape(ax.shape[0], -1, 32).max(-1), 32, axis=-1)
    half = 2.0 ** (-11 if f16 else -8) * 1.0001
    tiny = 2.0 ** -25 if f16 else 2.0 ** -133
    return half * np.abs(ref) + tiny + (x.shape[1] / 16 + 8) * 2.0 ** -23 * S + 2.0 ** -21 * (top @ aw.T)
