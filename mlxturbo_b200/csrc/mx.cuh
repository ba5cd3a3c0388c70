// mx.cuh -- the microscaled (MX) formats: blocks of 32 values along the last
// axis, each a small floating-point code times one power of two.
//
//   scale   2^e, stored as the byte e + 127 (ue8m0; 255 is NaN), with
//           e = floor(log2(max |v|)) - emax clamped to [-127, 127]
//   mxfp4   e2m1 codes (0 .5 1 1.5 2 3 4 6 and their negatives), emax = 2
//   mxfp8   e4m3 codes (largest 448, 0x7f / 0xff NaN), emax = 8
//   code    v * 2^-e rounded to nearest even, saturated
//
// the scale and rounding rule of the OCP Microscaling Formats specification
// v1.0 (section 6.3).  A block that holds an infinity or a NaN gets the scale
// byte 255: every value of it stands for NaN.
#pragma once

#include "common.cuh"

namespace qmm {

constexpr int MX_BLOCK = 32;

// What a tensor of values is made of.
enum MxType : int { MX_BF16 = QMM_BF16, MX_F16 = QMM_F16, MX_F32 = QMM_F32 };

// 2^(byte - 127) in fp32: exact for every byte (0 is the subnormal 2^-127, 255 NaN).
QMM_DEVINL float mx_scale_f32(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// The scale byte of a block from the bits of its largest |v| (fp32), and the
// factor 2^-e that brings the block onto the code grid (0 for a NaN block).
template <int EMAX>
QMM_DEVINL uint32_t mx_scale_byte(uint32_t amax_bits, float& inv) {
    const int b = (int)(amax_bits >> 23) - EMAX;
    const uint32_t byte = b > 0 ? (uint32_t)b : 0u;
    if (amax_bits >= 0x7F800000u) {
        inv = 0.0f;
        return 255u;
    }
    inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte), byte <= 254 - EMAX
    return byte;
}

QMM_DEVINL uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// Eight fp32 values to one word of e2m1 codes, the first in the low bits.
QMM_DEVINL uint32_t cvt8_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Two fp32 values to two e4m3 codes (a NaN becomes 0x7f).
QMM_DEVINL uint32_t cvt2_e4m3(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two e4m3 codes to two f16 values (exact).
QMM_DEVINL uint32_t e4m3x2_f16x2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}

// A word of eight e2m1 codes to four f16 pairs in order (exact).
QMM_DEVINL void e2m1x8_f16(uint32_t w, uint32_t (&p)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
        : "r"(w));
}

// Eight values of type T at p (16-byte aligned; fp32: two 16-byte loads) as fp32.
template <int T>
QMM_DEVINL void load8(const void* p, float (&v)[8]) {
    if constexpr (T == MX_F32) {
        const uint4 a = ld_v4(p), b = ld_v4(static_cast<const char*>(p) + 16);
        const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(u[j]);
    } else {
        using H = Half<T == MX_F16>;
        const uint4 a = ld_v4(p);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = H::lo_f32(u[j]);
            v[2 * j + 1] = H::hi_f32(u[j]);
        }
    }
}

template <int T>
QMM_DEVINL void store8(void* p, const float (&v)[8]) {
    uint4* o = static_cast<uint4*>(p);
    if constexpr (T == MX_F32) {
        o[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        o[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
        using H = Half<T == MX_F16>;
        o[0] = make_uint4(H::pack2(v[0], v[1]), H::pack2(v[2], v[3]), H::pack2(v[4], v[5]), H::pack2(v[6], v[7]));
    }
}

// Largest of the magnitudes of eight packed 16-bit floats, as one 16-bit
// pattern (patterns without the sign order like the magnitudes they stand for,
// infinity and then NaN above all), in both halves of the result's low bits.
QMM_DEVINL uint32_t max_abs8(const uint4& a) {
    const uint32_t M = 0x7FFF7FFFu;
    return __vmaxu2(__vmaxu2(a.x & M, a.y & M), __vmaxu2(a.z & M, a.w & M));
}
// The fp32 bits of the larger half.
template <bool F16>
QMM_DEVINL uint32_t max_abs_f32(uint32_t two) {
    const uint32_t m = max(two & 0xFFFFu, two >> 16);
    if constexpr (F16) return __float_as_uint(Half<true>::to_f32((uint16_t)m));
    else return m << 16;
}

// Four lanes of a warp hold a block, eight values each: to mxfp8, words and (by
// the first of the four) scale byte.  `o8` counts groups of
// eight values; lanes with `in` false only take part in the shuffles.
QMM_DEVINL void mx_store_block(const float (&v)[8], uint32_t* words, uint8_t* scales, long long o8, bool in) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float inv;
    const uint32_t byte = mx_scale_byte<8>(m, inv);
    if (!in) return;
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = byte == 255u ? 0.0f : v[j] * inv;
    const uint32_t lo = cvt2_e4m3(s[0], s[1]) | (cvt2_e4m3(s[2], s[3]) << 16);
    const uint32_t hi = cvt2_e4m3(s[4], s[5]) | (cvt2_e4m3(s[6], s[7]) << 16);
    reinterpret_cast<uint2*>(words)[o8] = make_uint2(lo, hi);
    if ((o8 & 3) == 0) scales[o8 >> 2] = (uint8_t)byte;
}

}  // namespace qmm

namespace qmm_host {

// One product with mxfp4 weights, dense or grouped by expert.
//   dense    y[m, :] = x[m, :] @ w^T, rows = M, E = 1, ids == nullptr
//   grouped  sorted row s (expert ids[s], ascending) takes x row
//            src ? src[s] : s and goes to y row dst ? dst[s] : s
struct MxMatmul {
    const void* x;            // bf16 / fp16 values, or e4m3 codes when xs is given
    const uint8_t* xs;        // scale bytes of x [x_rows, K/32], or null
    const uint32_t* w;        // [E, N, K/8]
    const uint8_t* ws;        // [E, N, K/32]
    void* y;                  // [rows, N]
    long long rows, x_rows, E, N, K;
    bool f16;                 // type of y (and of x when xs is null)
    const uint32_t* src;
    const uint32_t* dst;
    const int32_t* lhs;       // with it, x row lhs[src[s]] (the kernel of mx_f4.cu only)
    cudaStream_t st;
};
// The kernel for many rows, its rows per item and its workspace behind the row
// tables.
bool mx_tc_takes(long long rows, long long E, long long N, long long K);
int mx_tc_item_rows();
size_t mx_tc_workspace(long long rows, long long N, long long K, bool mx, bool f16, bool grouped);
int launch_mx_tc(const MxMatmul& a, const int4* items, const int32_t* n_items, const int32_t* ids, void* ws);
// The kernel for a few rows of an expert; item_rows 0 where it is not for this
// size.  items == nullptr in a grouped call (`ids` given):
// every row is an item of its own.
bool mx_f4_direct(long long rows, long long E, bool grouped);
bool mx_f4_takes(long long rows, long long E, long long N, long long K, bool mx, bool grouped);
int mx_f4_item_rows(long long rows, long long E, long long N, long long K, bool mx, bool grouped);
size_t mx_f4_workspace(long long rows, long long K, int bt);
int launch_mx_f4(const MxMatmul& a, const int4* items, const int32_t* n_items, const int32_t* ids, int bt, void* ws);
// Items (expert, first sorted row, rows) of at most ir rows from ascending ids,
// and their number; ids outside [0, E) have no item.
int launch_mx_items(const int32_t* ids_sorted, long long rows, int E, int ir, int32_t* row_start, int4* items,
                    long long items_max, int32_t* n_items, cudaStream_t st);
int launch_mx_quantize(const void* v, uint32_t* words, uint8_t* scales, long long n, int bits, int dtype,
                       cudaStream_t st);
int launch_mx_dequantize(const uint32_t* words, const uint8_t* scales, void* out, long long n, int bits, int dtype,
                         cudaStream_t st);
int launch_mx_rms_norm(const void* x, const void* residual, const void* weight, void* h, uint32_t* xq,
                       uint8_t* x_scales, long long rows, long long K, float eps, bool f16, cudaStream_t st);

}  // namespace qmm_host
