// mx_mma.cuh -- what the two block-scaled tensor-core kernels (mx_f4.cu,
// mx_tc.cu) share: bounded waits, scale bytes, signals between the blocks of a
// cluster, parameters.
#pragma once

#include "mx.cuh"
#include "tc.cuh"
#include "tma.cuh"

namespace qmm {

static __device__ int g_mx_error;  // one per translation unit

constexpr int MT_ROWS = 128;  // weight rows of a tile

// Bounded wait; false once it gave up, with the error flag set to `where` (the
// first wait of the kernel to give up).
// CLUSTER: acquires what other blocks of the cluster released.
template <bool CLUSTER = false>
QMM_DEVINL bool mt_wait(uint32_t bar, uint32_t parity, volatile int* abort, int where) {
    for (uint32_t i = 0; i < (1u << 22); ++i) {
        uint32_t ok;
        if constexpr (CLUSTER)
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(ok)
                : "r"(bar), "r"(parity)
                : "memory");
        else
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(ok)
                : "r"(bar), "r"(parity)
                : "memory");
        if (ok) return true;
        if ((i & 255u) == 255u && *abort) return false;
        if constexpr (CLUSTER) continue;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity), "r"(20u)
            : "memory");
        if (ok) return true;
    }
    *abort = 1;
    atomicCAS(&g_mx_error, 0, where);
    return false;
}

QMM_DEVINL uint32_t mt_cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The address of another block's shared memory.
QMM_DEVINL uint32_t mt_remote(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// An arrival there.  It orders this block's own memory only: what it announces
// is in its own shared memory behind a proxy fence, or is that it has read
// something.  (A cluster-wide release waits for every earlier store and costs
// about a microsecond.)
QMM_DEVINL void mt_pair_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// N floats stored there, counted on a barrier of the same block.
template <int N>
QMM_DEVINL void mt_remote_store(uint32_t addr, const float (&f)[N], uint32_t bar) {
    static_assert(N == 2 || N == 4, "one transaction");
    if constexpr (N == 4)
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                         addr),
                     "r"(__float_as_uint(f[0])), "r"(__float_as_uint(f[1])), "r"(__float_as_uint(f[2])),
                     "r"(__float_as_uint(f[3])), "r"(bar)
                     : "memory");
    else
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(
                         addr),
                     "r"(__float_as_uint(f[0])), "r"(__float_as_uint(f[1])), "r"(bar)
                     : "memory");
}
// All threads of the cluster; no memory is ordered by it (barriers are made
// visible by mbar_fence_init, everything else by mbarriers).
QMM_DEVINL void mt_cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
QMM_DEVINL void mt_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Scale bytes for one operand block of up to 128 rows x 4 blocks of 32 (512
// bytes): row r, block j at (r % 32) * 16 + (r / 32) * 4 + j.  Copied as 32
// lanes x 16 bytes to every lane quarter of four TMEM columns.
template <int CTAS = 1>
QMM_DEVINL void mt_copy_scales(uint32_t taddr, uint32_t saddr) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(128u >> 4) << 32;  // 8-row groups of 16-byte rows are 128 bytes apart
    d |= (uint64_t)1 << 46;
    if constexpr (CTAS == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

struct MxTcParams {
    const uint8_t* sfw;       // weight scale bytes [E * N, K/32]
    const uint8_t* sfb;       // plane scale bytes, rows of sfb_row
    const uint8_t *sfw_end, *sfb_end;
    uint16_t* y;
    const int4* items;        // grouped: (expert, first row, rows); dense: null
    const int32_t* n_items;
    const uint32_t* dst;      // y row of each row, or null
    int rows, N, K, KB;       // KB: k-blocks
    int n_tiles;              // weight tiles
    int sfb_row;              // K/32; of planes made here, that rounded up to 16, the rest zero
    int vec_w, vec_b;         // alignment of rows of scale bytes: 16, 4 or 1
};

struct MxTile {
    int expert, row0, rows, n0;
};

QMM_DEVINL void mt_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// The word at w (4-byte aligned); bytes outside of [lo, hi) are not read.
QMM_DEVINL uint32_t mt_word_within(const uint8_t* w, const uint8_t* lo, const uint8_t* hi) {
    if (w >= lo && w + 4 <= hi) return ld_dep(reinterpret_cast<const uint32_t*>(w));
    uint32_t v = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (w + c >= lo && w + c < hi) v |= (uint32_t)ld_dep(w + c) << (8 * c);
    return v;
}

// 16 bytes of a row of n scale bytes from `at`, those at or past n zero.  vec:
// every row starts on a multiple of so many bytes.  lo, hi: of the whole tensor.
// (Byte loads for vec = 1 held 16 rows of 6144x5152 at 36 us; 20 so.)
QMM_DEVINL uint4 mt_scale_bytes(const uint8_t* row, int at, int n, int vec, const uint8_t* lo, const uint8_t* hi) {
    if (vec == 16) return ld_v4(row + at);
    uint32_t w[4] = {};
    if (vec == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (at + 4 * c < n) w[c] = ld_dep(reinterpret_cast<const uint32_t*>(row + at) + c);
    } else {
        const uint32_t off = (uint32_t)(uintptr_t)(row + at) & 3u;
        const uint8_t* from = row + at - off;
        const int left = min(n - at, 16);
        uint32_t u[5];
#pragma unroll
        for (int c = 0; c < 5; ++c) u[c] = 4 * c < left + (int)off ? mt_word_within(from + 4 * c, lo, hi) : 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int k = left - 4 * c;
            w[c] = __funnelshift_r(u[c], u[c + 1], 8 * off) & (k >= 4 ? 0xFFFFFFFFu : k > 0 ? (1u << (8 * k)) - 1u : 0u);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace qmm

namespace qmm_host {

inline size_t mx_al256(size_t b) { return (b + 255) & ~(size_t)255; }

constexpr int kMxMaxBlocks = 148;

inline int mx_sm_count() {
    static int n = 0;
    if (!n) {
        int dev = 0, v = 0;
        if (cudaGetDevice(&dev) == cudaSuccess &&
            cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0)
            n = v < kMxMaxBlocks ? v : kMxMaxBlocks;
    }
    return n ? n : kMxMaxBlocks;
}

inline int mx_scale_vec(long long K, const void* a) {
    const uintptr_t both = (uintptr_t)a | (uintptr_t)(K / 32);
    return both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 1;
}

// Pitch of the scale bytes of planes: whole loads of 16 (512 rows of 6144x5152,
// where K/32 is odd: 44 us against 83 with byte-aligned rows).
inline long long mx_plane_row(long long K) { return (K / 32 + 15) & ~15LL; }

inline int mx_error_flag(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, qmm::g_mx_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int z = 0;
        cudaMemcpyToSymbol(qmm::g_mx_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace qmm_host
