// mx_tc.cu -- products of many rows with mxfp4 weights (prefill, large expert
// groups) on the block-scaled 8-bit tensor-core instruction
// (tcgen05.mma kind::mxf8f6f4), two SMs to a tile.
//
//   y[m, n] = sum_k w[n, k] * x[m, k],   w = e2m1 code * 2^e per 32 values
//
// The weights are the A operand: the instruction multiplies their codes and
// applies one scale byte per row and 32 values itself.  The B operand is e4m3.
// mxfp8 activations are that already.  A 16-bit activation is the sum of P
// e4m3 planes, each with its own block scale (mx_planes_kernel):
//
//   x = 2^e0 c0 + 2^(e0-4) c1 (+ 2^(e0-8) c2),  e0 = floor(log2 max|block|) - 7
//
// A code holds four significant bits, a plane four more than the one before, so
// two planes hold the 8 significant bits of bf16 and three the 11 of fp16,
// exactly, for values down to 2^-14 of the largest in their block of 32; below
// that the smallest code of the last plane leaves 2^-21 (bf16) or 2^-25 (fp16)
// of that largest value.
// The planes are further K of the same fp32 accumulator in TMEM.
//
// Bound by the tensor cores: 2 P M N K operations at the 8-bit rate, so a
// bf16 product runs at about the rate of a 16-bit one, without a weight ever
// being dequantised.  8192x17408x5120 takes 1052 us (bf16, 1.39 PFLOP/s of the
// product, 2.78 of the instruction), 1512 in fp16; 2011 rows of mxfp8 190 (1.9).
//
// A pair of blocks computes 256 weight rows x up to 192 activation rows; each
// holds its 128 weight rows and half of the activation rows in shared memory
// and its 128 rows of the sums in TMEM, twice, so that one tile's results are
// stored while the next is computed.  k-blocks of 128:
//   warp 0      TMA: packed weights and planes
//   warp 1      tensor memory; in the first block scale copies and MMAs
//   warps 2..9  two sets of four, a k-block each in turn: spread the weights'
//               codes, 8 to 16 bytes as the instruction reads them
//   warps 10..13 scale bytes into the instruction's layout
//   warps 14..17 epilogue: TMEM -> y
// TMA could spread the codes itself, but at 8 packed bytes a clock and SM: 1024
// clocks for 128 x 128, which the MMAs of one plane need 384 for.
//
// Pairs are persistent.  They take whole tiles, or, where there are fewer tiles than
// pairs, parts of one along K, which a second kernel adds.

#include "mx_mma.cuh"

namespace qmm {

constexpr int MT_BK = 128;   // K of a stage
constexpr int MT_BT = 192;   // activation rows of a tile
constexpr int MT_HALF = 96;  // of one block
constexpr int MT_W = 256;    // weight rows of a tile

QMM_DEVINL void mt_mma2(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// Arrive on this barrier of both blocks once the MMAs so far are done.
QMM_DEVINL void mt_commit2(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
// Instruction descriptor: A e2m1 (5), B e4m3 (0), both K-major, ue8m0 scales,
// 256 x N, scale byte `id` of the four in a TMEM column for both operands.
QMM_DEVINL uint32_t mt_idesc2(int N, uint32_t id) {
    return (id << 4) | (5u << 7) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(MT_W >> 7) << 27) | (id << 29);
}

struct MtParams {
    MxTcParams c;
    const int32_t* ids;   // grouped: expert of each y row
    int E;                // experts
    int split, part;      // parts of a tile along K, k-blocks of a part
    float* partial;       // split > 1: sums of the parts [split][rows][N]
};

// Every pairs-th tile, or part of one: k-blocks k0 .. k1 - 1, k0 a multiple of four.
struct MtWalk {
    uint32_t u, end, step;
    QMM_DEVINL MtWalk(uint32_t tiles, const MtParams& p)
        : u(blockIdx.x >> 1), end(tiles * (uint32_t)p.split), step(gridDim.x >> 1) {}
    QMM_DEVINL bool next(const MtParams& p, uint32_t& tile, int& k0, int& k1) {
        if (u >= end) return false;
        tile = u / (uint32_t)p.split;
        k0 = (int)(u - tile * (uint32_t)p.split) * p.part;
        k1 = min(p.c.KB, k0 + p.part);
        u += step;
        return true;
    }
};

QMM_DEVINL MxTile mt_tile(const MxTcParams& p, uint32_t tile) {
    MxTile t;
    const int item = (int)(tile / (uint32_t)p.n_tiles);
    t.n0 = ((int)tile - item * p.n_tiles) * MT_W;
    if (p.items) {
        const int4 it = ld_dep(p.items + item);
        t.expert = it.x;
        t.row0 = it.y;
        t.rows = it.z;
    } else {
        t.expert = 0;
        t.row0 = item * MT_BT;
        t.rows = min(MT_BT, p.rows - t.row0);
    }
    return t;
}

template <bool F16_, int P_, int STAGES_>
struct MxTc {
    static constexpr bool F16 = F16_;
    static constexpr int P = P_, STAGES = STAGES_;
    static constexpr int PACKS = 2;                     // ring of packed weights, two k-blocks each
    static constexpr int A_BYTES = MT_ROWS * MT_BK;     // spread
    static constexpr int PLANE = MT_HALF * MT_BK;
    static constexpr int B_BYTES = P * PLANE;
    static constexpr int S_BYTES = 512 * (1 + 2 * P);   // of a k-block: weights, then two blocks of columns per plane
    static constexpr int W_BYTES = MT_ROWS * MT_BK;     // packed, two k-blocks
    static constexpr int A_OFF = 0;
    static constexpr int B_OFF = A_OFF + STAGES * A_BYTES;
    static constexpr int W_OFF = B_OFF + STAGES * B_BYTES;
    static constexpr int SG = 2;                        // ring of scale groups, four k-blocks each
    static constexpr int S_OFF = W_OFF + PACKS * W_BYTES;
    static constexpr int BAR_OFF = S_OFF + SG * 4 * S_BYTES;
    static constexpr int BARS = 3 * STAGES + 2 * PACKS + 2 * SG + 4;
    static constexpr int SMEM = BAR_OFF + BARS * 8 + 32 + 1024;
    static constexpr int S_COLS = 4 * (1 + 2 * P);
    static constexpr int USED = 2 * MT_BT + STAGES * S_COLS;
    static constexpr int COLS = 512;
    static constexpr int THREADS = 576;
    static_assert(USED <= 512, "tensor memory");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
    mx_tc_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_b,
                 const MtParams p) {
    using H = Half<C::F16>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bars = sbase + C::BAR_OFF;
    auto full_b = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (STAGES + s); };
    auto ready = [&](int s) { return bars + 8 * (2 * STAGES + s); };  // of the first block
    auto full_w = [&](int w) { return bars + 8 * (3 * STAGES + w); };
    auto empty_w = [&](int w) { return bars + 8 * (3 * STAGES + C::PACKS + w); };
    auto scaled = [&](int g) { return bars + 8 * (3 * STAGES + 2 * C::PACKS + g); };  // of the first block
    auto s_empty = [&](int g) { return bars + 8 * (3 * STAGES + 2 * C::PACKS + C::SG + g); };
    auto acc_full = [&](int b) { return bars + 8 * (3 * STAGES + 2 * C::PACKS + 2 * C::SG + b); };
    auto acc_empty = [&](int b) { return bars + 8 * (3 * STAGES + 2 * C::PACKS + 2 * C::SG + 2 + b); };  // of the first
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + C::BARS * 8);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = mt_cluster_rank();
    if (threadIdx.x == 0) {
        *abort = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_b(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(ready(s), 8);
        }
        for (int w = 0; w < C::PACKS; ++w) {
            mbar_init(full_w(w), 1);
            mbar_init(empty_w(w), 8);
        }
        for (int g = 0; g < C::SG; ++g) {
            mbar_init(scaled(g), 8);
            mbar_init(s_empty(g), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 8);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tmap_w);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(C::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    mt_cluster_arrive();
    mt_cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t sf_cols = tmem + 2 * MT_BT;

    // Everything but the weights of a dense call may come from the kernel
    // before this one, so the other warps wait for it here, and the TMA warp
    // once the weights of its first ring are on the way.
    if (warp != 0 || p.c.items) pdl_wait();
    const uint32_t tiles =
        (uint32_t)p.c.n_tiles * (uint32_t)(p.c.items ? ld_dep(p.c.n_items) : (p.c.rows + MT_BT - 1) / MT_BT);
    MtWalk walk(tiles, p);
    uint32_t tile;
    int k0, k1;
    // columns of a tile's MMAs, and the first row of this block's half of them
    auto cols = [](const MxTile& t) { return max((t.rows + 31) & ~31, 32); };

    if (warp == 0) {
        // ---------------- TMA ----------------
        auto load_w = [&](const MxTile& t, int pair, int w) {
            mbar_expect_tx(full_w(w), C::W_BYTES);
            tma_load_2d(sbase + C::W_OFF + w * C::W_BYTES, &tmap_w, full_w(w), pair * MT_BK,
                        t.expert * p.c.N + t.n0 + (int)rank * MT_ROWS);
        };
        int i = 0, pack = 0, early = 0;  // k-blocks and pairs of them so far
        if (!p.c.items) {
            MtWalk ahead = walk;
            while (early < C::PACKS && ahead.next(p, tile, k0, k1)) {
                const MxTile t = mt_tile(p.c, tile);
                for (int j = k0 >> 1; 2 * j < k1 && early < C::PACKS; ++j, ++early)
                    if (elect_one()) load_w(t, j, early);
                __syncwarp();
            }
            pdl_wait();
        }
        while (walk.next(p, tile, k0, k1) && !*abort) {
            const MxTile t = mt_tile(p.c, tile);
            const int half = cols(t) / 2, mine = t.row0 + (int)rank * half;
            for (int kb = k0; kb < k1; ++kb, ++i) {
                if ((kb & 1) == 0) {
                    const int w = pack % C::PACKS;
                    if (pack >= early) {  // an early one may have been read and given back already
                        if (!mt_wait(empty_w(w), ((uint32_t)(pack / C::PACKS) & 1u) ^ 1u, abort, 64)) break;
                        if (elect_one()) load_w(t, kb >> 1, w);
                        __syncwarp();
                    }
                    ++pack;
                }
                const int s = i % STAGES;
                if (!mt_wait(empty(s), ((uint32_t)(i / STAGES) & 1u) ^ 1u, abort, 1)) break;
                const uint32_t b = sbase + C::B_OFF + s * C::B_BYTES;
                if (elect_one()) {
                    mbar_expect_tx(full_b(s), C::B_BYTES);
#pragma unroll
                    for (int q = 0; q < C::P; ++q)
                        tma_load_2d(b + q * C::PLANE, &tmap_b, full_b(s), kb * MT_BK, q * p.c.rows + mine);
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ---------------- scale copies and MMAs (first block) ----------------
        const uint64_t adesc0 = umma_desc_sw128(sbase + C::A_OFF), bdesc0 = umma_desc_sw128(sbase + C::B_OFF);
        int i = 0, seg = 0, g = -1;
        while (rank == 0 && walk.next(p, tile, k0, k1) && !*abort) {
            const int nb = cols(mt_tile(p.c, tile)), b = seg & 1;
            const uint32_t acc = tmem + b * MT_BT;
            if (!mt_wait(acc_empty(b), ((uint32_t)(seg >> 1) & 1u) ^ 1u, abort, 2)) break;
            ++seg;
            for (int kb = k0; kb < k1; ++kb, ++i) {
                const int s = i % STAGES;
                if ((kb & 3) == 0) {
                    ++g;
                    if (!mt_wait(scaled(g % C::SG), (uint32_t)(g / C::SG) & 1u, abort, 256)) break;
                }
                if (!mt_wait(ready(s), (uint32_t)(i / STAGES) & 1u, abort, 4)) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t sfa = sf_cols + s * C::S_COLS;
                    const uint32_t ssm = sbase + C::S_OFF + ((g % C::SG) * 4 + (kb & 3)) * C::S_BYTES;
#pragma unroll
                    for (int q = 0; q < 1 + 2 * C::P; ++q) mt_copy_scales<2>(sfa + 4 * q, ssm + 512 * q);
                    const uint64_t ad = adesc0 + ((uint32_t)(s * C::A_BYTES) >> 4);
                    const uint64_t bd = bdesc0 + ((uint32_t)(s * C::B_BYTES) >> 4);
#pragma unroll
                    for (int q = 0; q < C::P; ++q)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mt_mma2(acc, ad + 2 * j, bd + ((q * C::PLANE) >> 4) + 2 * j, mt_idesc2(nb, (uint32_t)j), sfa,
                                    sfa + 4 * (1 + 2 * q), kb != k0 || q || j);
                    mt_commit2(empty(s));
                    if ((kb & 3) == 3 || kb + 1 == k1) mt_commit2(s_empty(g % C::SG));
                }
                __syncwarp();
            }
            if (elect_one()) mt_commit2(acc_full(b));
            __syncwarp();
        }
    } else if (warp < 10) {
        // ---------------- codes ----------------
        // Thread r of a set has row r of this block's weights; set 0 takes the
        // even k-blocks, set 1 the odd.
        const int set = (warp - 2) >> 2, r = ((warp - 2) & 3) * 32 + lane;
        const uint32_t ready0 = mt_remote(ready(0), 0);
        int i0 = 0, pack = 0;  // k-blocks before this part, pairs so far
        while (walk.next(p, tile, k0, k1) && !*abort) {
            for (int j = k0 >> 1; 2 * j < k1; ++j, ++pack) {
                const int kb = 2 * j + set, w = pack % C::PACKS;
                const bool in = kb < k1;
                uint32_t c[4][4];
                if (!mt_wait(full_w(w), (uint32_t)(pack / C::PACKS) & 1u, abort, 8)) break;
                if (in) {
                    const uint32_t from = sbase + C::W_OFF + w * C::W_BYTES + r * 128;
#pragma unroll
                    for (int d = 0; d < 4; ++d)  // 128-byte swizzle: chunk ^ row
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(c[d][0]), "=r"(c[d][1]), "=r"(c[d][2]), "=r"(c[d][3])
                                     : "r"(from + (((4 * set + d) ^ (r & 7)) << 4))
                                     : "memory");
                }
                // the reads above come before TMA's next write to the buffer (an
                // arrive alone does not wait for them)
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(empty_w(w));
                if (!in) continue;
                const int i = i0 + kb - k0, s = i % STAGES;
                const uint32_t ph = (uint32_t)(i / STAGES) & 1u;
                if (!mt_wait(empty(s), ph ^ 1u, abort, 128)) break;
                const uint32_t to = sbase + C::A_OFF + s * C::A_BYTES + r * 128;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int e = 0; e < 2; ++e)  // 16 codes of 8 bytes to 16 bytes
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + (((2 * d + e) ^ (r & 7)) << 4)),
                                     "r"(c[d][2 * e]), "r"(c[d][2 * e + 1])
                                     : "memory");
                if (!mt_wait(full_b(s), ph, abort, 16)) break;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mt_pair_arrive(ready0 + 8 * s);
            }
            i0 += k1 - k0;
        }
    } else if (warp < 14) {
        // ---------------- scales ----------------
        // Thread r has row r of this block's weights, and columns r and r + 128
        // of the tile.  A group is 16 bytes of a row (four k-blocks); loads run
        // AHEAD groups ahead, across tiles.
        constexpr int NL = 1 + 2 * C::P;
        constexpr int AHEAD = C::P == 3 ? 2 : 3;
        const int r = (warp - 10) * 32 + lane, n_sf = p.c.K / 32;
        const uint32_t sdst = sbase + C::S_OFF + (r & 31) * 16 + (r >> 5) * 4;
        const uint32_t scaled0 = mt_remote(scaled(0), 0);
        const uint8_t* src[NL];
        int grp = 0, last = -1;
        bool more = true;
        auto enter = [&]() {  // the next part
            more = walk.next(p, tile, k0, k1);
            if (!more) return;
            const MxTile t = mt_tile(p.c, tile);
            src[0] = p.c.sfw + ((long long)t.expert * p.c.N + min(t.n0 + (int)rank * MT_ROWS + r, p.c.N - 1)) * n_sf;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = t.row0 + min(h * 128 + r, t.rows - 1);
#pragma unroll
                for (int q = 0; q < C::P; ++q) src[1 + 2 * q + h] = p.c.sfb + ((long long)q * p.c.rows + row) * p.c.sfb_row;
            }
            grp = k0 >> 2;
            last = (k1 - 1) >> 2;
        };
        auto load = [&](uint4 (&v)[NL]) {  // false past the end
            if (!more) return false;
            if (p.c.vec_w == 16 && p.c.vec_b == 16) {
                v[0] = ldg_v4(src[0] + 16 * grp);
#pragma unroll
                for (int q = 1; q < NL; ++q) v[q] = ld_v4(src[q] + 16 * grp);
            } else {
                v[0] = mt_scale_bytes(src[0], 16 * grp, n_sf, p.c.vec_w, p.c.sfw, p.c.sfw_end);
#pragma unroll
                for (int q = 1; q < NL; ++q)
                    v[q] = mt_scale_bytes(src[q], 16 * grp, n_sf, p.c.vec_b, p.c.sfb, p.c.sfb_end);
            }
            if (++grp > last) enter();
            return true;
        };
        uint4 v[AHEAD][NL];
        bool have[AHEAD];
        enter();
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) have[a] = load(v[a]);
        int g = 0;
        while (have[0] && !*abort) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (!have[a]) {
                    have[0] = false;
                    break;
                }
                if (!mt_wait(s_empty(g % C::SG), ((uint32_t)(g / C::SG) & 1u) ^ 1u, abort, 512)) break;
                const uint32_t to = sdst + (g % C::SG) * 4 * C::S_BYTES;
#pragma unroll
                for (int q = 0; q < NL; ++q) {
                    const uint32_t w[4] = {v[a][q].x, v[a][q].y, v[a][q].z, v[a][q].w};
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + c * C::S_BYTES + 512 * q), "r"(w[c])
                                     : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mt_pair_arrive(scaled0 + 8 * (g % C::SG));
                ++g;
                have[a] = load(v[a]);
            }
        }
    } else {
        // ---------------- epilogue ----------------
        const int quarter = warp & 3, row = quarter * 32 + lane;  // weight row of the block = TMEM lane
        const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
        if (p.ids)  // y rows whose id has no expert
            for (int q = blockIdx.x * 4 + warp - 14; q < p.c.rows; q += gridDim.x * 4)
                if ((uint32_t)ld_dep(p.ids + q) >= (uint32_t)p.E)
                    for (int n = lane; n < p.c.N; n += 32) p.c.y[(long long)q * p.c.N + n] = 0;
        const uint32_t acc_empty0 = mt_remote(acc_empty(0), 0);
        int seg = 0;
        while (walk.next(p, tile, k0, k1) && !*abort) {
            const MxTile t = mt_tile(p.c, tile);
            const int b = seg & 1;
            if (!mt_wait(acc_full(b), (uint32_t)(seg >> 1) & 1u, abort, 32)) break;
            ++seg;
            tc_fence_after();
            const int n = t.n0 + (int)rank * MT_ROWS + row;
            // Two lanes exchange halves, so that each stores two neighbouring
            // outputs at once: the even lane for even rows, the odd for odd.
            const bool pairs = (p.c.N & 1) == 0;
            const int n2 = n & ~1;
#pragma unroll 1
            for (int c0 = 0; c0 < t.rows; c0 += 32) {
                uint32_t u[32];
                tmem_ld32(t_lane + b * MT_BT + c0, u);
                int out_l = t.row0 + c0 + lane;  // y row of column c0 + lane
                if (p.c.dst && c0 + lane < t.rows) out_l = (int)ld_dep(p.c.dst + out_l);
                tmem_wait_ld();
                if (p.split > 1) {  // 128 bytes of a row to a warp
                    float* part = p.partial + ((long long)(k0 / p.part) * p.c.rows + t.row0 + c0) * p.c.N + n;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c0 + j < t.rows && n < p.c.N) part[(long long)j * p.c.N] = __uint_as_float(u[j]);
                } else if (pairs) {
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const uint32_t mine = lane & 1 ? u[j + 1] : u[j], give = lane & 1 ? u[j] : u[j + 1];
                        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 1);
                        const uint32_t lo = lane & 1 ? got : mine, hi = lane & 1 ? mine : got;
                        const int out = __shfl_sync(0xffffffffu, out_l, j + (lane & 1));
                        if (c0 + j + (lane & 1) < t.rows && n2 < p.c.N)
                            *reinterpret_cast<uint32_t*>(p.c.y + (long long)out * p.c.N + n2) =
                                H::pack2(__uint_as_float(lo), __uint_as_float(hi));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const long long out = __shfl_sync(0xffffffffu, out_l, j);
                        if (c0 + j < t.rows && n < p.c.N) p.c.y[out * p.c.N + n] = H::from_f32(__uint_as_float(u[j]));
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mt_pair_arrive(acc_empty0 + 8 * b);
        }
    }
    if (p.split > 1) pdl_launch_dependents();
    if (*abort) __nanosleep(1000000);  // after a wait gave up: let copies in flight land
    tc_fence_before();
    __syncwarp();
    // a block's shared memory outlives the other's last access to it
    mt_cluster_arrive();
    mt_cluster_wait();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
    }
}

// y = the sum of a divided product's parts, in their order; four values to a thread.
template <bool F16>
__global__ void __launch_bounds__(256) mx_join_kernel(const float* partial, uint16_t* y, long long n, int split) {
    using H = Half<F16>;
    constexpr int RUN = 4;  // loads together
    pdl_wait();
    for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 4; i < n;
         i += (long long)gridDim.x * blockDim.x * 4) {
        float f[4] = {};
        for (int s0 = 0; s0 < split; s0 += RUN) {
            float v[RUN][4];
#pragma unroll
            for (int s = 0; s < RUN; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[s][j] = 0.0f;
#pragma unroll
            for (int s = 0; s < RUN; ++s) {
                if (s0 + s >= split) continue;
                const float* from = partial + (s0 + s) * n + i;
                if ((n & 3) == 0) {
                    const uint4 w = ld_v4(from);
                    v[s][0] = __uint_as_float(w.x), v[s][1] = __uint_as_float(w.y);
                    v[s][2] = __uint_as_float(w.z), v[s][3] = __uint_as_float(w.w);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (i + j < n) v[s][j] = ld_dep(from + j);
                }
            }
#pragma unroll
            for (int s = 0; s < RUN; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] += v[s][j];
        }
        if ((n & 3) == 0) {
            *reinterpret_cast<uint2*>(y + i) = make_uint2(H::pack2(f[0], f[1]), H::pack2(f[2], f[3]));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < n) y[i + j] = H::from_f32(f[j]);
        }
    }
}

// The two planes of bf16 rows, sixteen values to a thread, two at a time in
// bf16, where a power of two, the cut after four bits and the remainder are
// exact.  False (for the warp) where a block holds a value below the smallest
// normal code or one that is not finite.
QMM_DEVINL bool mt_planes_bf16(const uint4 (&raw)[2], bool live, uint4 (&out)[2], uint32_t& byte) {
    const uint32_t u[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
    uint32_t m = max_abs_f32<false>(__vmaxu2(max_abs8(raw[0]), max_abs8(raw[1])));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    float inv;
    byte = mx_scale_byte<7>(m, inv);
    const uint32_t inv2 = (__float_as_uint(inv) >> 16) * 0x10001u;
    uint32_t v2[8], least = 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(v2[j]) : "r"(u[j]), "r"(inv2));
        least = __vminu2(least, v2[j] & 0x7FFF7FFFu);
    }
    const bool plain = byte >= 4 && m < 0x7F800000u && (least & 0xFFFFu) >= 0x3C80u && (least >> 16) >= 0x3C80u;  // 2^-6
    if (!__all_sync(0xffffffffu, plain || !live)) return false;
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t top = v2[j] & 0xFFF0FFF0u;
        uint32_t minus, rest;  // 16 (v - top)
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(minus) : "r"(top), "r"(0xC180C180u));
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(rest) : "r"(v2[j]), "r"(0x41804180u), "r"(minus));
        hi[j] = cvt2_e4m3(Half<false>::lo_f32(top), Half<false>::hi_f32(top));
        lo[j] = cvt2_e4m3(Half<false>::lo_f32(rest), Half<false>::hi_f32(rest));
    }
    out[0] = make_uint4(hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16), hi[4] | (hi[5] << 16), hi[6] | (hi[7] << 16));
    out[1] = make_uint4(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16), lo[4] | (lo[5] << 16), lo[6] | (lo[7] << 16));
    return true;
}

// Eight values of either 16-bit type to P planes, given their block's largest
// finite magnitude.
template <int T, int P>
QMM_DEVINL void mt_planes8(const uint4& raw, uint32_t block_max, uint2 (&out)[P], uint32_t (&bytes)[P]) {
    using H = Half<T == MX_F16>;
    float v[8] = {H::lo_f32(raw.x), H::hi_f32(raw.x), H::lo_f32(raw.y), H::hi_f32(raw.y),
                  H::lo_f32(raw.z), H::hi_f32(raw.z), H::lo_f32(raw.w), H::hi_f32(raw.w)};
    float inv;
    // 128 <= largest < 256 on the grid: rounding cannot reach 448
    uint32_t byte = mx_scale_byte<7>(block_max, inv);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        v[j] = abs_bits(v[j]) < 0x7F800000u ? v[j] * inv : __uint_as_float(0x7FC00000u);  // an infinity has no code
#pragma unroll
    for (int q = 0; q < P; ++q) {
        // what this plane's code holds: the first four significant bits, or
        // whole units of 2^-9 below the smallest normal code
        float code[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float four = __uint_as_float(__float_as_uint(v[j]) & 0xFFF00000u);
            const float unit = __fsub_rn(__fadd_rn(v[j], 24576.0f), 24576.0f);
            code[j] = q + 1 == P ? v[j] : fabsf(v[j]) < 0x1p-6f ? unit : four;
        }
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = cvt2_e4m3(code[2 * j], code[2 * j + 1]);
        out[q] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        bytes[q] = byte;
        const uint32_t next = byte > 4 ? byte - 4 : 0;  // the remainder, up to 16 times larger
        const float up = __uint_as_float((127u + byte - next) << 23);
        byte = next;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (v[j] - code[j]) * up;
    }
}
// Largest finite magnitude of eight values, as fp32 bits.
template <bool F16>
QMM_DEVINL uint32_t mt_max_finite(const uint4& raw) {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    constexpr uint32_t INF = F16 ? 0x7C00u : 0x7F80u;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = u[j] & 0x7FFFu, b = (u[j] >> 16) & 0x7FFFu;
        m = max(m, max(a < INF ? a : 0u, b < INF ? b : 0u));
    }
    return max_abs_f32<F16>(m);
}

// Activations to P e4m3 planes [P][R][K] with scales [P][R][K/32 rounded
// up to 16], rows taken through src; two lanes hold a block.  P = 1 copies mxfp8 rows.
template <int T, int P>
__global__ void __launch_bounds__(128) mx_planes_kernel(const void* x, const uint8_t* xs, uint8_t* planes,
                                                        uint8_t* scales, const uint32_t* src, int x_rows, int R,
                                                        int K) {
    pdl_launch_dependents();
    // sixteen values (half a block) of RUN rows to a thread, their loads together
    constexpr int RUN = 4;
    const int g = K / 16, c = blockIdx.x * blockDim.x + threadIdx.x;
    const bool in = c < g;  // whole blocks of 32 are in or out
    const long long plane = (long long)R * g;
    const int n_sf = K / 32, pitch = (n_sf + 15) & ~15;
    // scale byte of plane q of a row's block, by the first lane of two; the last block's clears the rest of the row
    auto put_scale = [&](int q, long long row, uint32_t byte) {
        if (c & 1) return;
        uint8_t* to = scales + ((long long)q * R + row) * pitch;
        to[c >> 1] = (uint8_t)byte;
        if (c + 2 == g) {
#pragma unroll 1
            for (int j = n_sf; j < pitch; ++j) to[j] = 0;
        }
    };
    for (int r0 = blockIdx.y * RUN; r0 < R; r0 += gridDim.y * RUN) {
        long long from[RUN];
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            const int r = min(r0 + k, R - 1);
            from[k] = r;
            if (src) {
                from[k] = ld_dep(src + r);
                from[k] = from[k] < x_rows ? from[k] : x_rows - 1;
            }
        }
        constexpr int NV = P == 1 ? 1 : 2;
        uint4 raw[RUN][2];
        uint32_t e[RUN];
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
#pragma unroll
            for (int d = 0; d < NV; ++d)
                raw[k][d] = in ? ld_v4(static_cast<const uint4*>(x) + (from[k] * g + c) * NV + d) : make_uint4(0, 0, 0, 0);
            if constexpr (P == 1) e[k] = in && (c & 1) == 0 ? ld_dep(xs + from[k] * (K / 32) + (c >> 1)) : 0;
        }
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            const long long i = (long long)(r0 + k) * g + c;
            const bool live = in && r0 + k < R;
            uint4* out = reinterpret_cast<uint4*>(planes) + i;
            if constexpr (P == 1) {
                if (!live) continue;
                out[0] = raw[k][0];
                put_scale(0, r0 + k, e[k]);
            } else {
                if constexpr (T == MX_BF16) {
                    uint4 two[2];
                    uint32_t byte;
                    if (mt_planes_bf16(raw[k], live, two, byte)) {
                        if (!live) continue;
                        out[0] = two[0];
                        out[plane] = two[1];
                        put_scale(0, r0 + k, byte);
                        put_scale(1, r0 + k, byte - 4);
                        continue;
                    }
                }
                uint32_t m = max(mt_max_finite<T == MX_F16>(raw[k][0]), mt_max_finite<T == MX_F16>(raw[k][1]));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                uint2 lo[P], hi[P];
                uint32_t bytes[P];
                mt_planes8<T, P>(raw[k][0], m, lo, bytes);
                mt_planes8<T, P>(raw[k][1], m, hi, bytes);
                if (!live) continue;
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    out[q * plane] = make_uint4(lo[q].x, lo[q].y, hi[q].x, hi[q].y);
                    put_scale(q, r0 + k, bytes[q]);
                }
            }
        }
    }
}

}  // namespace qmm

namespace qmm_host {

namespace {

// Workspace of a product behind the row tables.
struct TcLayout {
    size_t planes, scales, partial, bytes;
};

int planes_of(bool mx, bool f16) { return mx ? 1 : f16 ? 3 : 2; }

long long tc_tiles_max(long long rows, long long E, long long N, bool grouped) {
    const long long bt = qmm::MT_BT;
    const long long items = grouped ? rows / bt + (E < rows ? E : rows) + 1 : (rows + bt - 1) / bt;
    return items * ((N + qmm::MT_W - 1) / qmm::MT_W);
}

// Parts of a tile along K: as many as leave no pair idle, each of at least 8
// k-blocks, in dense products.  Their sums meet in fp32 in the workspace, added
// by mx_join_kernel.  (bf16, 512 rows of 1024x5120: 24 us, 27 a tile's whole K
// alone.  Stretches of equal length over tile ends, with the parts added by the
// pair that came last: 54 us, 128 rows of 17408x5120 52 against 31.)
struct TcSplit {
    int split, part;
};
TcSplit tc_split(long long rows, long long N, long long K, bool grouped) {
    const long long tiles = tc_tiles_max(rows, 1, N, false), KB = (K + 127) / 128;
    long long s = grouped ? 1 : kMxMaxBlocks / 2 / tiles;
    s = s > KB / 8 ? KB / 8 : s;
    if (s < 2) return {1, (int)KB};
    const long long part = ((KB + s - 1) / s + 3) / 4 * 4;  // whole groups of scale bytes
    return {(int)((KB + part - 1) / part), (int)part};
}

// planes: of every row of the product; mxfp8 rows that are taken in order are
// read where they are
TcLayout tc_layout(long long rows, long long N, long long K, bool mx, bool f16, bool grouped) {
    TcLayout l{};
    const int P = planes_of(mx, f16);
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t o = at;
        at += mx_al256(n);
        return o;
    };
    l.planes = take(mx && !grouped ? 0 : (size_t)P * rows * K);
    l.scales = take(mx && !grouped ? 0 : (size_t)P * rows * mx_plane_row(K));
    const TcSplit d = tc_split(rows, N, K, grouped);
    l.partial = take(d.split > 1 ? (size_t)d.split * rows * N * 4 : 0);
    l.bytes = at;
    return l;
}

template <class C>
int launch_tc(const MxMatmul& a, const CUtensorMap& mw, const CUtensorMap& mb, const qmm::MtParams& p, int pairs,
              bool pdl) {
    auto kern = qmm::mx_tc_kernel<C>;
    int rc = ensure_smem_limit((const void*)kern, C::SMEM, "mx_tc smem attribute");
    if (rc) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = a.st;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl && pdl_enabled() ? 2 : 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kern, mw, mb, p), "mx_tc launch");
}

}  // namespace

int mx_tc_item_rows() { return qmm::MT_BT; }

bool mx_tc_takes(long long rows, long long E, long long N, long long K) {
    return E * N <= (1LL << 31) - 512 && 3 * rows <= (1LL << 31) - 512 &&
           tc_tiles_max(rows, E, N, true) * ((K + 127) / 128) < (1LL << 31);
}

size_t mx_tc_workspace(long long rows, long long N, long long K, bool mx, bool f16, bool grouped) {
    return tc_layout(rows, N, K, mx, f16, grouped).bytes;
}

int launch_mx_tc(const MxMatmul& a, const int4* items, const int32_t* n_items, const int32_t* ids, void* ws) {
    const bool mx = a.xs != nullptr, grouped = items != nullptr, in_place = mx && !a.src;
    const int P = planes_of(mx, a.f16);
    const TcLayout l = tc_layout(a.rows, a.N, a.K, mx, a.f16, grouped);
    char* const base = static_cast<char*>(ws);
    const long long tiles = tc_tiles_max(a.rows, a.E, a.N, grouped);
    uint8_t* planes = reinterpret_cast<uint8_t*>(base + l.planes);
    uint8_t* scales = reinterpret_cast<uint8_t*>(base + l.scales);
    qmm::MtParams p{};
    p.c.sfw = a.ws;
    p.c.sfb = in_place ? a.xs : scales;
    p.c.y = static_cast<uint16_t*>(a.y);
    p.c.items = items;
    p.c.n_items = n_items;
    p.c.dst = a.dst;
    p.c.rows = (int)a.rows;
    p.c.N = (int)a.N;
    p.c.K = (int)a.K;
    p.c.KB = (int)((a.K + 127) / 128);
    p.c.n_tiles = (int)((a.N + qmm::MT_W - 1) / qmm::MT_W);
    p.c.sfw_end = a.ws + a.E * a.N * (a.K / 32);
    p.c.sfb_row = (int)(in_place ? a.K / 32 : mx_plane_row(a.K));
    p.c.sfb_end = p.c.sfb + P * (in_place ? a.x_rows : a.rows) * p.c.sfb_row;
    p.c.vec_w = mx_scale_vec(a.K, a.ws);
    p.c.vec_b = in_place ? mx_scale_vec(a.K, a.xs) : 16;
    p.ids = ids;
    p.E = (int)a.E;
    const TcSplit d = tc_split(a.rows, a.N, a.K, grouped);
    p.split = d.split;
    p.part = d.part;
    p.partial = reinterpret_cast<float*>(base + l.partial);
    const int most = mx_sm_count() / 2;
    const long long pairs = tiles * d.split < most ? tiles * d.split : most;

    int rc = QMM_OK;
    if (!in_place) {
        const int g = (int)(a.K / 16);
        const long long runs = (a.rows + 3) / 4;
        const dim3 grid((unsigned)((g + 127) / 128), (unsigned)(runs < 32768 ? runs : 32768));
#define QMM_PLANES(T, PP)                                                                                         \
    qmm::mx_planes_kernel<T, PP><<<grid, 128, 0, a.st>>>(a.x, a.xs, planes, scales, a.src, (int)a.x_rows,          \
                                                         (int)a.rows, (int)a.K)
        if (mx) QMM_PLANES(qmm::MX_BF16, 1);
        else if (a.f16) QMM_PLANES(qmm::MX_F16, 3);
        else QMM_PLANES(qmm::MX_BF16, 2);
#undef QMM_PLANES
        rc = cuda_status(cudaGetLastError(), "mx_planes launch");
    }
    if (rc) return rc;
    CUtensorMap mw, mb;
    rc = tensor_map_2d(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, (uint64_t)a.K / 2, (uint64_t)(a.E * a.N),
                       (uint64_t)a.K / 2, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = tensor_map_2d(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, in_place ? a.x : planes, (uint64_t)a.K,
                       (uint64_t)(P * a.rows), (uint64_t)a.K, 128, qmm::MT_HALF, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    using namespace qmm;
    if (mx) rc = a.f16 ? launch_tc<MxTc<true, 1, 6>>(a, mw, mb, p, (int)pairs, !in_place)
                       : launch_tc<MxTc<false, 1, 6>>(a, mw, mb, p, (int)pairs, !in_place);
    else rc = a.f16 ? launch_tc<MxTc<true, 3, 3>>(a, mw, mb, p, (int)pairs, true)
                    : launch_tc<MxTc<false, 2, 4>>(a, mw, mb, p, (int)pairs, true);
    if (rc || d.split == 1) return rc;
    const long long n = a.rows * a.N, blocks = (n + 1023) / 1024;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(blocks < 2 * kMxMaxBlocks ? blocks : 2 * kMxMaxBlocks));
    cfg.blockDim = dim3(256);
    cfg.stream = a.st;
    cudaLaunchAttribute at[1]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, a.f16 ? mx_join_kernel<true> : mx_join_kernel<false>,
                                          (const float*)p.partial, p.c.y, n, d.split),
                       "mx_join launch");
}

int mx_tc_device_error(int reset) { return mx_error_flag(reset); }

}  // namespace qmm_host
