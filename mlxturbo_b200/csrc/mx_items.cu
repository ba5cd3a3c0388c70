// mx_items.cu -- row tables of a product grouped by expert whose ids come sorted:
// which expert, from which row and how many rows each tile takes.

#include "mx.cuh"

namespace qmm {

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
// rows, never a row or an item out of range: row_start may then go up and down
// as its writers happened to finish, up to rows / ir items for every expert, which
// 32 bits do not hold.
__global__ void __launch_bounds__(1024) mx_items_kernel(const int32_t* row_start, int E, int ir, int4* items,
                                                        int items_max, int32_t* n_items) {
    __shared__ long long wsum[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (E + (int)blockDim.x - 1) / (int)blockDim.x;
    const int e0 = min(E, (int)threadIdx.x * per), e1 = min(E, e0 + per);
    long long n = 0;
    for (int e = e0; e < e1; ++e) n += (max(0, ld_dep(row_start + e + 1) - ld_dep(row_start + e)) + ir - 1) / ir;
    long long inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        long long s = wsum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        wsum[lane] = s;
    }
    __syncthreads();
    long long at = inc - n + (warp ? wsum[warp - 1] : 0);
    for (int e = e0; e < e1; ++e) {
        const int a = ld_dep(row_start + e), b = ld_dep(row_start + e + 1);
        for (int r = a; r < b && at < items_max; r += ir) items[at++] = make_int4(e, r, min(ir, b - r), 0);
    }
    if (threadIdx.x == 0) *n_items = (int)min(wsum[31], (long long)items_max);
}

}  // namespace qmm

namespace qmm_host {

int launch_mx_items(const int32_t* ids_sorted, long long rows, int E, int ir, int32_t* row_start, int4* items,
                    long long items_max, int32_t* n_items, cudaStream_t st) {
    qmm::mx_row_start_kernel<<<(unsigned)(rows / 256 + 1), 256, 0, st>>>(ids_sorted, (int)rows, E, row_start);
    const int rc = cuda_status(cudaGetLastError(), "mx_row_start launch");
    if (rc) return rc;
    qmm::mx_items_kernel<<<1, 1024, 0, st>>>(row_start, E, ir, items, (int)items_max, n_items);
    return cuda_status(cudaGetLastError(), "mx_items launch");
}

}  // namespace qmm_host
