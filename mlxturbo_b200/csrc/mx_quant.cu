// mx_quant.cu -- values to and from the microscaled formats, and the residual
// norm that writes mxfp8 rows.
//
// Replaces mx.quantize / mx.dequantize with mode="mxfp4" / "mxfp8" (the
// reference calls them in affine mode only, mlxturbo/rebit.py:103-121).

#include "mx.cuh"

namespace qmm {

// A block of 32 values sits in four lanes, eight values (one 16-byte load of a
// 16-bit type) each; rows are whole blocks, so the tensor is a flat run of
// blocks.  Bound by HBM: 2 + 17/32 (mxfp4) or 2 + 33/32 (mxfp8) bytes a value
// for 16-bit inputs.
template <int T, int BITS>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const void* v, uint32_t* words, uint8_t* scales,
                                                          long long n8) {
    constexpr int SZ = T == MX_F32 ? 32 : 16;  // bytes of eight values
    const long long step = (long long)gridDim.x * blockDim.x;
    // whole warps stay in the loop: the shuffles need every lane
    for (long long base = ((long long)blockIdx.x * blockDim.x + threadIdx.x) & ~31LL; base < n8; base += step) {
        const long long i = base + (threadIdx.x & 31);
        const bool in = i < n8;
        float f[8] = {};
        if (in) load8<T>(static_cast<const char*>(v) + i * SZ, f);
        mx_store_block<BITS>(f, words, scales, i, in);
    }
}

// One thread for eight codes.  The product of a code and its scale is exact in
// fp32 (at most four significant bits; 2^-127 times a code is a subnormal fp32)
// and is rounded once, to the output type.
template <int T, int BITS>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint32_t* words, const uint8_t* scales, void* out,
                                                            long long n8) {
    constexpr int SZ = T == MX_F32 ? 32 : 16;
    const long long step = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += step) {
        const float s = mx_scale_f32(ld_dep(scales + (i >> 2)));
        uint32_t p[4];
        if constexpr (BITS == 4) {
            e2m1x8_f16(ld_dep(words + i), p);
        } else {
            const uint2 w = ld_dep(reinterpret_cast<const uint2*>(words) + i);
            p[0] = e4m3x2_f16x2(w.x & 0xFFFFu);
            p[1] = e4m3x2_f16x2(w.x >> 16);
            p[2] = e4m3x2_f16x2(w.y & 0xFFFFu);
            p[3] = e4m3x2_f16x2(w.y >> 16);
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

// s = x + residual (fp32), h = s rounded to the 16-bit type,
// y = s / sqrt(mean(s^2) + eps) * weight, written as mxfp8.
//
// blockDim.x threads (a multiple of 32) share a row, blockDim.y rows a block; a
// thread keeps VPT groups of eight values of the row in registers between the
// sum of squares and the normalisation, so x and the residual are read once.
// VPT = 0 (rows too long for that) reads them again.  Sums in fp32, in an order
// that depends on the row length only.
template <bool F16, int VPT, bool RES>
__global__ void __launch_bounds__(1024) mx_rms_norm_kernel(const uint16_t* x, const uint16_t* res, const uint16_t* weight, uint16_t* h,
                                   uint32_t* xq, uint8_t* xs, long long rows, int n8, float eps) {
    constexpr int T = F16 ? MX_F16 : MX_BF16;
    constexpr int V = VPT ? VPT : 1;
    __shared__ float part[2][32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const float inv_k = 1.0f / (8.0f * (float)n8);
    int flip = 0;
    for (long long r0 = (long long)blockIdx.x * blockDim.y; r0 < rows; r0 += (long long)gridDim.x * blockDim.y) {
        const long long row = r0 + threadIdx.y;
        const bool live = row < rows;
        const long long first = row * n8;
        float v[V][8];
        float sq = 0.0f;
        auto load = [&](int i, float (&f)[8]) {
            load8<T>(x + (first + i) * 8, f);
            if constexpr (RES) {
                float g[8];
                load8<T>(res + (first + i) * 8, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] += g[j];
            }
        };
        const int groups = VPT ? VPT : (n8 + blockDim.x - 1) / blockDim.x;
#pragma unroll
        for (int a = 0; a < groups; ++a) {
            const int i = threadIdx.x + a * blockDim.x;
            float(&f)[8] = v[VPT ? a : 0];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = 0.0f;
            if (live && i < n8) {
                load(i, f);
                if constexpr (RES) store8<T>(h + (first + i) * 8, f);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(f[j], f[j], sq);
        }
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
            mx_store_block<8>(f, xq, xs, first + i, in);
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
    const long long n8 = n / 8;
    if (n8 == 0) return QMM_OK;
    const unsigned g = mx_grid(n8);
#define QMM_MX(T)                                                                                     \
    (bits == 4 ? qmm::mx_quantize_kernel<T, 4><<<g, 256, 0, st>>>(v, words, scales, n8)               \
               : qmm::mx_quantize_kernel<T, 8><<<g, 256, 0, st>>>(v, words, scales, n8))
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
    int vpt = n8 <= 1024 ? 1 : n8 <= 2048 ? 2 : n8 <= 4096 ? 4 : 0;
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
