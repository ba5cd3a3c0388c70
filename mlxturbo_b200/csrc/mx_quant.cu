// mx_quant.cu -- values to and from the microscaled formats, and the residual
// norm that writes mxfp8 rows.
//
// Replaces mx.quantize / mx.dequantize with mode="mxfp4" / "mxfp8" (the
// reference calls them in affine mode only, mlxturbo/rebit.py:103-121).

#include "mx.cuh"

namespace qmm {

// Half a block of 32 values to a thread; rows are whole blocks, so the tensor
// is a flat run of blocks.  Bound by HBM: 2 + 17/32 (mxfp4) or 2 + 33/32
// (mxfp8) bytes a value for 16-bit inputs.  UNROLL halves of a thread are
// loaded together: with one, 17408x5120 bf16 to mxfp4 took 51 us; with two, there
// and back (mx_dequantize_kernel) takes 80, 451 MB at 5.6 TB/s.
template <int T, int BITS>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const void* v, uint32_t* words, uint8_t* scales,
                                                          long long n16) {
    constexpr int UNROLL = T == MX_F32 ? 1 : 2;
    constexpr int NV = T == MX_F32 ? 4 : 2;  // 16-byte loads of a half
    const long long span = (long long)gridDim.x * blockDim.x;
    const uint4* in = static_cast<const uint4*>(v);
    // whole warps stay in the loop: the shuffles need every lane
    for (long long base = ((long long)blockIdx.x * blockDim.x + threadIdx.x) & ~31LL; base < n16;
         base += UNROLL * span) {
        uint4 raw[UNROLL][NV];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
            const long long i = base + k * span + (threadIdx.x & 31);
#pragma unroll
            for (int d = 0; d < NV; ++d) raw[k][d] = i < n16 ? ld_v4(in + i * NV + d) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
            const long long i = base + k * span + (threadIdx.x & 31);
            float f[16];
            uint32_t m = 0;
            if constexpr (T == MX_F32) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t u[4] = {raw[k][d].x, raw[k][d].y, raw[k][d].z, raw[k][d].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[4 * d + j] = __uint_as_float(u[j]);
                        m = max(m, u[j] & 0x7FFFFFFFu);
                    }
                }
            } else {
                using H = Half<T == MX_F16>;
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    const uint32_t u[4] = {raw[k][d].x, raw[k][d].y, raw[k][d].z, raw[k][d].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[8 * d + 2 * j] = H::lo_f32(u[j]);
                        f[8 * d + 2 * j + 1] = H::hi_f32(u[j]);
                    }
                }
                m = max_abs_f32<T == MX_F16>(__vmaxu2(max_abs8(raw[k][0]), max_abs8(raw[k][1])));
            }
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            float inv;
            const uint32_t byte = mx_scale_byte<BITS == 4 ? 2 : 8>(m, inv);
            if (i >= n16) continue;
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] = byte == 255u ? 0.0f : f[j] * inv;
            if constexpr (BITS == 4) {
                const float lo[8] = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
                const float hi[8] = {f[8], f[9], f[10], f[11], f[12], f[13], f[14], f[15]};
                reinterpret_cast<uint2*>(words)[i] = make_uint2(cvt8_e2m1(lo), cvt8_e2m1(hi));
            } else {
                uint32_t w[4];
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    w[d] = cvt2_e4m3(f[4 * d], f[4 * d + 1]) | (cvt2_e4m3(f[4 * d + 2], f[4 * d + 3]) << 16);
                reinterpret_cast<uint4*>(words)[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if ((i & 1) == 0) scales[i >> 1] = (uint8_t)byte;
        }
    }
}

// Eight codes to a thread, so that a warp's stores are contiguous.  The product
// of a code and its scale is exact in fp32 (at most four significant bits;
// 2^-127 times a code is a subnormal fp32) and is rounded once, to the output
// type.
template <int T, int BITS>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint32_t* words, const uint8_t* scales, void* out,
                                                            long long n8) {
    constexpr int SZ = T == MX_F32 ? 32 : 16;  // bytes of eight values
    constexpr int UNROLL = 4;
    const long long span = (long long)gridDim.x * blockDim.x;
    for (long long base = (long long)blockIdx.x * blockDim.x + threadIdx.x; base < n8; base += UNROLL * span) {
        uint2 w[UNROLL];
        uint32_t byte[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
            const long long i = base + k * span;
            w[k] = make_uint2(0, 0);
            byte[k] = 0;
            if (i >= n8) continue;
            byte[k] = ld_dep(scales + (i >> 2));
            if constexpr (BITS == 4) w[k].x = ld_dep(words + i);
            else w[k] = ld_dep(reinterpret_cast<const uint2*>(words) + i);
        }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
            const long long i = base + k * span;
            if (i >= n8) continue;
            const float s = mx_scale_f32(byte[k]);
            uint32_t p[4];
            if constexpr (BITS == 4) {
                e2m1x8_f16(w[k].x, p);
            } else {
                p[0] = e4m3x2_f16x2(w[k].x & 0xFFFFu);
                p[1] = e4m3x2_f16x2(w[k].x >> 16);
                p[2] = e4m3x2_f16x2(w[k].y & 0xFFFFu);
                p[3] = e4m3x2_f16x2(w[k].y >> 16);
            }
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[2 * j] = Half<true>::lo_f32(p[j]) * s;
                f[2 * j + 1] = Half<true>::hi_f32(p[j]) * s;
            }
            store8<T>(static_cast<char*>(out) + i * SZ, f);
        }
    }
}

// s = x + residual (fp32), h = s rounded to the 16-bit type,
// y = s / sqrt(mean(s^2) + eps) * weight, written as mxfp8.
//
// blockDim.x threads (a multiple of 32) share a row, blockDim.y rows a block; a
// thread keeps VPT groups of eight values of the row in registers between the
// sum of squares and the normalisation, so x and the residual are read once,
// and has the next row's on the way meanwhile.  VPT = 0 (rows too long for
// that) reads them again.  Sums in fp32, in an order that depends on the row
// length only.  Bound by HBM: 6 + 33/32 bytes a value; with the mxfp8 rows
// dequantised again, 8192x5120 takes 70 us, 422 MB at 6.0 TB/s.
template <bool F16, int VPT, bool RES>
__global__ void __launch_bounds__(1024) mx_rms_norm_kernel(const uint16_t* x, const uint16_t* res,
                                                           const uint16_t* weight, uint16_t* h, uint32_t* xq,
                                                           uint8_t* xs, long long rows, int n8, float eps) {
    constexpr int T = F16 ? MX_F16 : MX_BF16;
    constexpr int V = VPT ? VPT : 1;
    using H = Half<F16>;
    __shared__ float part[2][32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const float inv_k = 1.0f / (8.0f * (float)n8);
    const long long step = (long long)gridDim.x * blockDim.y;
    uint4 nx[V], nr[V];  // the next row's x and residual
    auto fetch = [&](long long row) {
#pragma unroll
        for (int a = 0; a < V; ++a) {
            const int i = threadIdx.x + a * blockDim.x;
            nx[a] = nr[a] = make_uint4(0, 0, 0, 0);
            if (row < rows && i < n8) {
                nx[a] = ld_v4(x + (row * n8 + i) * 8);
                if constexpr (RES) nr[a] = ld_v4(res + (row * n8 + i) * 8);
            }
        }
    };
    auto widen = [&](const uint4& p, const uint4& q, float (&f)[8]) {
        const uint32_t u[4] = {p.x, p.y, p.z, p.w}, w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = H::lo_f32(u[j]);
            f[2 * j + 1] = H::hi_f32(u[j]);
            if constexpr (RES) {
                f[2 * j] += H::lo_f32(w[j]);
                f[2 * j + 1] += H::hi_f32(w[j]);
            }
        }
    };
    int flip = 0;
    long long r0 = (long long)blockIdx.x * blockDim.y;
    if constexpr (VPT > 0) fetch(r0 + threadIdx.y);
    for (; r0 < rows; r0 += step) {
        const long long row = r0 + threadIdx.y;
        const bool live = row < rows;
        const long long first = row * n8;
        float v[V][8];
        float sq = 0.0f;
        auto load = [&](int i, float (&f)[8]) {  // rows too long for registers
            const uint4 p = ld_v4(x + (first + i) * 8);
            uint4 q = make_uint4(0, 0, 0, 0);
            if constexpr (RES) q = ld_v4(res + (first + i) * 8);
            widen(p, q, f);
        };
        const int groups = VPT ? VPT : (n8 + blockDim.x - 1) / blockDim.x;
#pragma unroll
        for (int a = 0; a < groups; ++a) {
            const int i = threadIdx.x + a * blockDim.x;
            const bool in = live && i < n8;
            float(&f)[8] = v[VPT ? a : 0];
            if constexpr (VPT > 0) {
                widen(nx[a], nr[a], f);  // zeros outside
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = 0.0f;
                if (in) load(i, f);
            }
            if constexpr (RES)
                if (in) store8<T>(h + (first + i) * 8, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(f[j], f[j], sq);
        }
        if constexpr (VPT > 0) fetch(row + step);
#pragma unroll
        for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        if (warps > 1) {
            if (lane == 0) part[flip][threadIdx.y][warp] = sq;
            __syncthreads();
            sq = lane < warps ? part[flip][threadIdx.y][lane] : 0.0f;
#pragma unroll
            for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
            flip ^= 1;
        }
        const float rstd = __frsqrt_rn(fmaf(sq, inv_k, eps));
#pragma unroll
        for (int a = 0; a < groups; ++a) {
            const int i = threadIdx.x + a * blockDim.x;
            const bool in = live && i < n8;
            float(&f)[8] = v[VPT ? a : 0];
            if constexpr (VPT == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = 0.0f;
                if (in) load(i, f);
            }
            float g[8] = {};
            if (in) load8<T>(weight + (long long)i * 8, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = f[j] * rstd * g[j];
            mx_store_block(f, xq, xs, first + i, in);
        }
    }
}

}  // namespace qmm

namespace qmm_host {

static unsigned mx_grid(long long threads) {
    const long long b = (threads + 255) / 256;
    return (unsigned)(b < 148 * 8 ? b : 148 * 8);
}

int launch_mx_quantize(const void* v, uint32_t* words, uint8_t* scales, long long n, int bits, int dtype,
                       cudaStream_t st) {
    const long long n16 = n / 16;
    if (n16 == 0) return QMM_OK;
    const unsigned g = mx_grid(n16);
#define QMM_MX(T)                                                                                     \
    (bits == 4 ? qmm::mx_quantize_kernel<T, 4><<<g, 256, 0, st>>>(v, words, scales, n16)               \
               : qmm::mx_quantize_kernel<T, 8><<<g, 256, 0, st>>>(v, words, scales, n16))
    if (dtype == qmm::MX_BF16) QMM_MX(qmm::MX_BF16);
    else if (dtype == qmm::MX_F16) QMM_MX(qmm::MX_F16);
    else QMM_MX(qmm::MX_F32);
#undef QMM_MX
    return cuda_status(cudaGetLastError(), "mx_quantize launch");
}

int launch_mx_dequantize(const uint32_t* words, const uint8_t* scales, void* out, long long n, int bits, int dtype,
                         cudaStream_t st) {
    const long long n8 = n / 8;
    if (n8 == 0) return QMM_OK;
    const unsigned g = mx_grid(n8);
#define QMM_MX(T)                                                                                     \
    (bits == 4 ? qmm::mx_dequantize_kernel<T, 4><<<g, 256, 0, st>>>(words, scales, out, n8)           \
               : qmm::mx_dequantize_kernel<T, 8><<<g, 256, 0, st>>>(words, scales, out, n8))
    if (dtype == qmm::MX_BF16) QMM_MX(qmm::MX_BF16);
    else if (dtype == qmm::MX_F16) QMM_MX(qmm::MX_F16);
    else QMM_MX(qmm::MX_F32);
#undef QMM_MX
    return cuda_status(cudaGetLastError(), "mx_dequantize launch");
}

int launch_mx_rms_norm(const void* x, const void* residual, const void* weight, void* h, uint32_t* xq,
                       uint8_t* x_scales, long long rows, long long K, float eps, bool f16, cudaStream_t st) {
    if (rows == 0) return QMM_OK;
    const int n8 = (int)(K / 8);
    // by the row length alone, which fixes the order of the sums
    const int vpt = n8 <= 256 ? 1 : n8 <= 2048 ? 2 : n8 <= 4096 ? 4 : 0;
    const int per = vpt ? (n8 + vpt - 1) / vpt : 1024;
    const int tx = (per + 31) / 32 * 32;
    int ty = 256 / tx;  // short rows: several to a block
    if (ty < 1) ty = 1;
    if (ty > rows) ty = (int)rows;
    const long long blocks = (rows + ty - 1) / ty, most = 148LL * (2048 / (tx * ty));
    const dim3 grid((unsigned)(blocks < most ? blocks : most)), block(tx, ty);
#define QMM_MX(F, V)                                                                                              \
    (residual ? qmm::mx_rms_norm_kernel<F, V, true><<<grid, block, 0, st>>>(                                       \
                    static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),                       \
                    static_cast<const uint16_t*>(weight), static_cast<uint16_t*>(h), xq, x_scales, rows, n8, eps)  \
              : qmm::mx_rms_norm_kernel<F, V, false><<<grid, block, 0, st>>>(                                      \
                    static_cast<const uint16_t*>(x), nullptr, static_cast<const uint16_t*>(weight), nullptr, xq,   \
                    x_scales, rows, n8, eps))
#define QMM_MXV(F) (vpt == 1 ? QMM_MX(F, 1) : vpt == 2 ? QMM_MX(F, 2) : vpt == 4 ? QMM_MX(F, 4) : QMM_MX(F, 0))
    if (f16) QMM_MXV(true);
    else QMM_MXV(false);
#undef QMM_MXV
#undef QMM_MX
    return cuda_status(cudaGetLastError(), "mx_rms_norm launch");
}

}  // namespace qmm_host
