// mx_warp.cu -- products with mxfp4 weights on warp-level matrix instructions,
// for every width that is a whole number of blocks (K % 32 == 0); and the row
// tables of the grouped form.
//
//   y[m, n] = sum over blocks b of 2^(ew[n,b]) * sum_{k in b} code(w[n,k]) * x[m,k]
//
// The e2m1 codes become bf16 (or fp16) exactly, a block is two m16n8k16
// instructions into a zero accumulator, and the block's scale (times the
// activation's, when x is mxfp8) enters as one fp32 multiply-add per output.
//
// A thread of the fragment layout owns columns 2t, 2t+1, 2t+8, 2t+9 of each of
// the two instructions.  The order of k inside a block is free as long as both
// operands agree, so it takes k = 8t .. 8t+7 of the block instead: one packed
// word of weights and one 16-byte load of activations, with nothing moved
// between lanes.
//
// RG row groups of 16 weight rows times KW shares of K make the eight warps of
// a block; with KW > 1 the shares are added in shared memory in warp order.

#include "mx.cuh"

namespace qmm {

template <bool F16>
QMM_DEVINL uint32_t f16x2_to(uint32_t p) {
    if constexpr (F16) return p;
    // e2m1 value in f16 -> bf16: exponent field moved down three bits, then
    // times 2^112 (the difference of the biases), exact
    const uint32_t r = ((p >> 3) & 0x0FFF0FFFu) | (p & 0x80008000u);
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(r), "r"(0x77807780u));
    return d;
}

// XQ: x is mxfp8 (multiplied as fp16); else x has the output type.
template <bool F16, bool XQ, int NT, int KW>
__global__ void __launch_bounds__(256) mx_warp_kernel(const void* x, const uint8_t* xs, const uint32_t* w,
                                                      const uint8_t* ws, uint16_t* y, int M, int N, int K, int x_rows,
                                                      const int4* items, const int32_t* n_items, const uint32_t* src,
                                                      const uint32_t* dst) {
    using H = Half<F16>;
    constexpr bool MF16 = F16 || XQ;  // operand type of the matrix instructions
    constexpr int RG = 8 / KW;
    __shared__ float red[KW > 1 ? 8 * 16 * NT * 8 : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int kw = warp % KW, rg = warp / KW;
    const int G = K / 32;
    int expert = 0;
    long long row0 = (long long)blockIdx.y * (NT * 8);
    int rows = M - (int)row0;
    if (items) {
        if ((int)blockIdx.y >= ld_dep(n_items)) return;
        const int4 it = ld_dep(items + blockIdx.y);
        expert = it.x;
        row0 = it.y;
        rows = it.z;
    }
    if (rows > NT * 8) rows = NT * 8;
    const int n_a = (blockIdx.x * RG + rg) * 16 + g, n_b = n_a + 8;
    const long long wa_row = (long long)expert * N + min(n_a, N - 1), wb_row = (long long)expert * N + min(n_b, N - 1);
    const uint32_t* wa = w + wa_row * (G * 4) + t;
    const uint32_t* wb = w + wb_row * (G * 4) + t;
    const uint8_t* sa = ws + wa_row * G;
    const uint8_t* sb = ws + wb_row * G;
    // activation rows of this thread: column g of each token tile (operand), columns 2t, 2t+1 (scales)
    auto x_row = [&](int j) -> int {
        long long s = row0 + min(j, rows - 1);
        if (src) s = ld_dep(src + s);
        return (int)(s < x_rows ? s : x_rows - 1);
    };
    int xr[NT], xc[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        xr[i] = x_row(i * 8 + g);
        if constexpr (XQ) {
            xc[i][0] = x_row(i * 8 + 2 * t);
            xc[i][1] = x_row(i * 8 + 2 * t + 1);
        }
    }
    float acc[NT][4] = {};
    const float zero[4] = {};
    const int b0 = (int)((long long)G * kw / KW), b1 = (int)((long long)G * (kw + 1) / KW);
#pragma unroll 2
    for (int b = b0; b < b1; ++b) {
        uint32_t pa[4], pb[4];
        e2m1x8_f16(wa[b * 4], pa);
        e2m1x8_f16(wb[b * 4], pb);
        const float s_a = mx_scale_f32(sa[b]), s_b = mx_scale_f32(sb[b]);
        uint32_t a[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            a[j][0] = f16x2_to<MF16>(pa[2 * j]);
            a[j][1] = f16x2_to<MF16>(pb[2 * j]);
            a[j][2] = f16x2_to<MF16>(pa[2 * j + 1]);
            a[j][3] = f16x2_to<MF16>(pb[2 * j + 1]);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            uint4 v;
            float s0 = 1.0f, s1 = 1.0f;
            if constexpr (XQ) {
                const uint2 q = ld_dep(reinterpret_cast<const uint2*>(
                    static_cast<const uint8_t*>(x) + (long long)xr[i] * K + b * 32 + 8 * t));
                v = make_uint4(e4m3x2_f16x2(q.x & 0xFFFFu), e4m3x2_f16x2(q.x >> 16), e4m3x2_f16x2(q.y & 0xFFFFu),
                               e4m3x2_f16x2(q.y >> 16));
                s0 = mx_scale_f32(ld_dep(xs + (long long)xc[i][0] * G + b));
                s1 = mx_scale_f32(ld_dep(xs + (long long)xc[i][1] * G + b));
            } else {
                v = ld_v4(static_cast<const uint16_t*>(x) + (long long)xr[i] * K + b * 32 + 8 * t);
            }
            float p[4];
            mma16816<MF16>(p, a[0], v.x, v.y, zero);
            mma16816<MF16>(p, a[1], v.z, v.w, p);
            if constexpr (XQ) {
                // activation scale first: both products of powers of two could
                // leave the fp32 range only together
                p[0] *= s0;
                p[1] *= s1;
                p[2] *= s0;
                p[3] *= s1;
            }
            acc[i][0] = fmaf(s_a, p[0], acc[i][0]);
            acc[i][1] = fmaf(s_a, p[1], acc[i][1]);
            acc[i][2] = fmaf(s_b, p[2], acc[i][2]);
            acc[i][3] = fmaf(s_b, p[3], acc[i][3]);
        }
    }
    if constexpr (KW > 1) {
        float* mine = red + warp * (16 * NT * 8);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[(i * 4 + j) * 32 + lane] = acc[i][j];
        __syncthreads();
        if (kw != 0) return;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float s = acc[i][j];
                for (int q = 1; q < KW; ++q) s += mine[q * (16 * NT * 8) + (i * 4 + j) * 32 + lane];
                acc[i][j] = s;
            }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int j = i * 8 + 2 * t + c;
            if (j >= rows) continue;
            const long long out = dst ? (long long)ld_dep(dst + row0 + j) : row0 + j;
            uint16_t* yr = y + out * N;
            if (n_a < N) yr[n_a] = H::from_f32(acc[i][c]);
            if (n_b < N) yr[n_b] = H::from_f32(acc[i][2 + c]);
        }
}

// Ascending ids -> first row of each expert: a row whose id differs from its
// predecessor's starts every expert between the two.
__global__ void __launch_bounds__(256) mx_row_start_kernel(const int32_t* ids, int rows, int E, int32_t* row_start) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i > rows) return;
    const int lo = i == 0 ? -1 : max(-1, min(E, ld_dep(ids + i - 1)));
    const int hi = i == rows ? E : max(-1, min(E, ld_dep(ids + i)));
    for (int e = lo + 1; e <= hi; ++e) row_start[e] = i;
}

// Items of at most ir rows from the experts' first rows: their numbers per
// expert, prefix-summed over one block.  Ids that were not ascending give wrong
// rows, never a row or an item out of range.
__global__ void __launch_bounds__(1024) mx_items_kernel(const int32_t* row_start, int E, int ir, int4* items,
                                                        int items_max, int32_t* n_items) {
    __shared__ int wsum[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (E + (int)blockDim.x - 1) / (int)blockDim.x;
    const int e0 = min(E, (int)threadIdx.x * per), e1 = min(E, e0 + per);
    int n = 0;
    for (int e = e0; e < e1; ++e) n += (max(0, ld_dep(row_start + e + 1) - ld_dep(row_start + e)) + ir - 1) / ir;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int s = wsum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        wsum[lane] = s;
    }
    __syncthreads();
    int at = inc - n + (warp ? wsum[warp - 1] : 0);
    for (int e = e0; e < e1; ++e) {
        const int a = ld_dep(row_start + e), b = ld_dep(row_start + e + 1);
        for (int r = a; r < b && at < items_max; r += ir) items[at++] = make_int4(e, r, min(ir, b - r), 0);
    }
    if (threadIdx.x == 0) *n_items = min(wsum[31], items_max);
}

__global__ void mx_zero_rows_kernel(const int32_t* ids, int rows, int E, uint16_t* y, long long N) {
    const int r = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (r >= rows || (uint32_t)ld_dep(ids + r) < (uint32_t)E) return;
    for (long long n = threadIdx.x & 31; n < N; n += 32) y[r * N + n] = 0;
}

}  // namespace qmm

namespace qmm_host {

template <bool F16, bool XQ, int NT, int KW>
static int launch_warp(const MxMatmul& a, const int4* items, const int32_t* n_items, long long gy) {
    const int rows_per = 16 * (8 / KW);
    if (gy > 65535) {
        set_error("mxfp4 product: %lld row tiles of %d (limit 65535)", gy, NT * 8);
        return QMM_EUNSUPPORTED;
    }
    const dim3 grid((unsigned)((a.N + rows_per - 1) / rows_per), (unsigned)gy);
    qmm::mx_warp_kernel<F16, XQ, NT, KW><<<grid, 256, 0, a.st>>>(
        a.x, a.xs, a.w, a.ws, static_cast<uint16_t*>(a.y), (int)a.rows, (int)a.N, (int)a.K, (int)a.x_rows, items,
        n_items, a.src, a.dst);
    return cuda_status(cudaGetLastError(), "mx_warp launch");
}

template <bool F16, bool XQ>
static int launch_warp_tile(const MxMatmul& a, const int4* items, const int32_t* n_items, long long items_max,
                            int item_rows) {
    const long long gy = items ? items_max : (a.rows + item_rows - 1) / item_rows;
    if (item_rows == 8) return launch_warp<F16, XQ, 1, 8>(a, items, n_items, gy);
    if (item_rows == 16) return launch_warp<F16, XQ, 2, 8>(a, items, n_items, gy);
    return launch_warp<F16, XQ, 8, 1>(a, items, n_items, gy);
}

// Up to 16 rows of an expert share one pass over its weights with K divided
// among the warps; more rows take 64 at a time, weight rows divided instead.
int mx_warp_item_rows(long long rows, long long E) {
    const long long mean = (rows + E - 1) / E;
    return mean <= 8 ? 8 : mean <= 16 ? 16 : 64;
}

int launch_mx_warp(const MxMatmul& a, const int4* items, const int32_t* n_items, long long items_max, int item_rows) {
    if (a.xs) {
        return a.f16 ? launch_warp_tile<true, true>(a, items, n_items, items_max, item_rows)
                     : launch_warp_tile<false, true>(a, items, n_items, items_max, item_rows);
    }
    return a.f16 ? launch_warp_tile<true, false>(a, items, n_items, items_max, item_rows)
                 : launch_warp_tile<false, false>(a, items, n_items, items_max, item_rows);
}

int launch_mx_items(const int32_t* ids_sorted, long long rows, int E, int ir, int32_t* row_start, int4* items,
                    long long items_max, int32_t* n_items, cudaStream_t st) {
    qmm::mx_row_start_kernel<<<(unsigned)(rows / 256 + 1), 256, 0, st>>>(ids_sorted, (int)rows, E, row_start);
    const int rc = cuda_status(cudaGetLastError(), "mx_row_start launch");
    if (rc) return rc;
    qmm::mx_items_kernel<<<1, 1024, 0, st>>>(row_start, E, ir, items, (int)items_max, n_items);
    return cuda_status(cudaGetLastError(), "mx_items launch");
}

int launch_mx_zero_rows(const int32_t* ids, long long rows, int E, void* y, long long N, cudaStream_t st) {
    qmm::mx_zero_rows_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(ids, (int)rows, E,
                                                                          static_cast<uint16_t*>(y), N);
    return cuda_status(cudaGetLastError(), "mx_zero_rows launch");
}

}  // namespace qmm_host
