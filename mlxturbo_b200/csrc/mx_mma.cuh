// mx_mma.cuh -- what the two block-scaled tensor-core kernels (mx_f4.cu,
// mx_tc.cu) share: bounded waits, scale copies, the division of the work over
// persistent blocks and the joining of divided tiles.
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
    const uint8_t* sfb;       // plane scale bytes, rows of K/32
    uint16_t* y;
    const int4* items;        // grouped: (expert, first row, rows); dense: null
    const int32_t* n_items;
    const uint32_t* dst;      // y row of each row, or null
    float* partial;           // split: parts of tiles
    uint32_t* counters;       // split: one per tile and 32 weight rows, zero
    int rows, N, K, KB;       // KB: k-blocks
    int n_tiles, split;
    int vec;                  // bytes that one load of scale bytes may take: 16, 4 or 1
};

// The stretches of k-blocks of one tile that worker `me` of `count` (a pair of
// blocks) has, in order.  Whole tiles: every count-th.  Split: of g workers the
// first `more` have base + 1 k-blocks and the others base, consecutive.  32-bit arithmetic: the
// host keeps tiles * KB below 2^31.
struct MxWalk {
    uint32_t u, end, kb, step;
    uint32_t base, more;
    QMM_DEVINL MxWalk(const MxTcParams& p, uint32_t tiles, uint32_t me, uint32_t count) : kb((uint32_t)p.KB) {
        if (p.split) {
            const uint32_t all = tiles * kb, g = min(all, count);  // a worker with no k-block shares nothing
            step = base = more = u = end = 0;
            if (g) {
                base = all / g;
                more = all - base * g;
            }
            if (me < g) {
                u = start_of(me);
                end = start_of(me + 1);
            }
        } else {
            base = more = 0;
            step = count;
            u = me;
            end = tiles;
        }
    }
    QMM_DEVINL uint32_t start_of(uint32_t block) const { return block * base + min(block, more); }
    QMM_DEVINL uint32_t block_of(uint32_t unit) const {
        const uint32_t big = more * (base + 1);
        return unit < big ? unit / (base + 1) : more + (unit - big) / base;
    }
    QMM_DEVINL bool next(uint32_t& tile, int& k0, int& k1) {
        if (u >= end) return false;
        if (step) {
            tile = u;
            k0 = 0;
            k1 = (int)kb;
            u += step;
        } else {
            tile = u / kb;
            k0 = (int)(u - tile * kb);
            k1 = (int)min(kb, (uint32_t)k0 + (end - u));
            u += (uint32_t)(k1 - k0);
        }
        return true;
    }
};

struct MxTile {
    int expert, row0, rows, n0;
};
QMM_DEVINL MxTile mt_tile(const MxTcParams& p, uint32_t tile, int bt, int weight_rows) {
    MxTile t;
    const int item = (int)(tile / (uint32_t)p.n_tiles);
    t.n0 = ((int)tile - item * p.n_tiles) * weight_rows;
    if (p.items) {
        const int4 it = ld_dep(p.items + item);
        t.expert = it.x;
        t.row0 = it.y;
        t.rows = it.z;
    } else {
        t.expert = 0;
        t.row0 = item * bt;
        t.rows = min(bt, p.rows - t.row0);
    }
    return t;
}

QMM_DEVINL void mt_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// 16 scale bytes of a row from `at`, bytes at or past `n` zero.
QMM_DEVINL uint4 mt_scale_bytes(const uint8_t* row, int at, int n, int vec) {
    if (vec == 16) return ld_v4(row + at);
    uint32_t w[4] = {};
    if (vec == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (at + 4 * c < n) w[c] = ld_dep(reinterpret_cast<const uint32_t*>(row + at) + c);
    } else {
#pragma unroll
        for (int c = 0; c < 16; ++c)
            if (at + c < n) w[c >> 2] |= (uint32_t)ld_dep(row + at + c) << (8 * (c & 3));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A worker that computed a part of a tile stored it in its slot; true for the
// warp that has to join the parts (of its 32 weight rows, with a counter of
// their own): the last of the workers first .. final that share the tile.
QMM_DEVINL bool mt_last_of(const MxWalk& w, uint32_t tile, uint32_t* counter, int& first, int& final_) {
    first = (int)w.block_of(tile * w.kb);
    final_ = (int)w.block_of(tile * w.kb + w.kb - 1);
    __threadfence();
    __syncwarp();
    uint32_t before = 0;
    if ((threadIdx.x & 31) == 0) before = atomicAdd(counter, 1u);
    if (__shfl_sync(0xffffffffu, before, 0) != (uint32_t)(final_ - first)) return false;
    __threadfence();
    return true;
}

// The parts of eight columns (128 rows each, from `base` of the first worker's
// slots), added in the order of k.  Slot 0 of a worker is a stretch that begins
// inside a tile (its first), slot 1 one that begins with the tile and ends
// inside it (its last).
QMM_DEVINL void mt_join8(const float* base, long long slot, int first, int final_, int nj, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.0f;
    for (int c = first; c <= final_; c += 4) {
        float v[4][8];  // loads of four workers in flight
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const float* from = base + (2 * (c + d) + (c + d == first)) * slot;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[d][j] = c + d <= final_ && j < nj ? __ldcg(from + j * MT_ROWS) : 0.0f;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] += v[d][j];
    }
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

inline int mx_scale_vec(long long K, const void* a, const void* b) {
    const uintptr_t both = (uintptr_t)a | (uintptr_t)b | (uintptr_t)(K / 32);
    return both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 1;
}

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
