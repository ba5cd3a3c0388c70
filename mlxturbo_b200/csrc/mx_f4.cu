// mx_f4.cu -- products of a few rows with mxfp4 weights (decode, verify, small
// expert groups) on the 4-bit tensor-core instruction (tcgen05.mma kind::mxf4).
//
// Bound by the weight stream: 17/32 byte a weight.  The instruction takes both
// operands as packed e2m1 codes with a ue8m0 scale per 32, so the weights go
// from HBM through TMA to the tensor core exactly as stored, with no unpacking
// anywhere.  An activation becomes eight signed octal digits,
//
//   x = 2^e * sum over q < 8 of 8^-q * d_q / 2,   d_q in -4 .. 3,
//   2^e > max|block| >= 2^(e-1)
//
// d/2 is an e2m1 value and 2^e 8^-q a block scale, so digit q of every value
// makes one e2m1 plane.  Eight digits are a 24-bit fixed-point number: an
// activation is held to 2^-22 of the largest of its block of 32 (bf16 exactly
// down to 2^-14 of it, fp16 to 2^-11, an e4m3 block exactly).  Products and
// sums are fp32 in TMEM, where a plane is a column; the epilogue adds the
// eight, small ones first.  A block below 2^-103 is held to 2^-126, the smallest
// scale's limit; one with an infinity or a NaN, or with an mxfp8 value of 2^128
// or more, makes its row NaN.  The first plane's sum may be twice the whole, so
// results of 2^127 and above may become infinite.
//
// 5 rows of 17408x5120 (47 MB) take 13.9 us, 1 of 248320x5120 (675 MB) 115 us,
// 5.9 TB/s: start and end of the launch, and the kernel that makes the planes,
// cost every call the same.
//
// Eight-bit planes (mx_tc.cu) were tried here first: they need the codes spread
// to bytes in shared memory, and TMA spreads 8 packed bytes a clock and SM,
// which held 17408x5120 (47 MB) at 24 us.
//
// One block, k-blocks of 256 in a ring:
//   warp 0        TMA: weights (and planes, where a kernel before made them)
//   warp 1        tensor memory, scale copies, MMAs
//   warps 2..5    weight scale bytes into the instruction's layout
//   warps 6..9    epilogue
//   warps 10..25  up to two rows: activations to digits, straight into the
//                 operand's layout in shared memory
// S blocks of a cluster share a tile, each with its part of K; the first adds
// the others' sums from its shared memory in the order of k.  Clusters are
// persistent over tiles.

#include <cmath>

#include "mx_mma.cuh"
#include "mx_ring.cuh"

namespace qmm {

constexpr int F4_BK = 256;  // K of a stage: 128 bytes of a row
constexpr int F4_PLANES = 8;
constexpr int F4_FIRST = 3;  // k-blocks of weights asked for before the first activations are in

enum F4X : int { F4_BF16 = 0, F4_FP16 = 1, F4_MX8 = 2, F4_PLANED = 3 };

// A and B e2m1, both K-major, ue8m0 scales; K = 64: the two scale bytes at
// `id` (0 or 2) of a TMEM column for both operands.
QMM_DEVINL constexpr uint32_t f4_idesc(int N, uint32_t id) {
    return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) |
           ((uint32_t)(MT_ROWS >> 7) << 27) | (id << 29);
}

QMM_DEVINL void f4_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// Eight activations of four lanes' block of 32 as fp32, and the scale byte of
// the block's first plane (255: not a number) with the factor to 2^22 units.
// twice: the block reaches 2^127 and 2^128 is no scale.  Its digits are those of
// half the values, the first plane's codes those of d instead of d / 2, the other
// planes' scales one up.
struct F4Group {
    float v[8];
    uint32_t byte;
    float mul;
    bool twice;
};

template <int X>
QMM_DEVINL F4Group f4_group(uint4 raw, uint32_t mx_byte) {
    F4Group g;
    uint32_t m = 0;
    if constexpr (X == F4_MX8) {
        const uint32_t h[4] = {e4m3x2_f16x2(raw.x & 0xFFFFu), e4m3x2_f16x2(raw.x >> 16), e4m3x2_f16x2(raw.y & 0xFFFFu),
                               e4m3x2_f16x2(raw.y >> 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            g.v[2 * j] = Half<true>::lo_f32(h[j]);
            g.v[2 * j + 1] = Half<true>::hi_f32(h[j]);
            m = max(m, max(abs_bits(g.v[2 * j]), abs_bits(g.v[2 * j + 1])));
        }
    } else {
        using H = Half<X == F4_FP16>;
        const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            g.v[2 * j] = H::lo_f32(u[j]);
            g.v[2 * j + 1] = H::hi_f32(u[j]);
            m = max(m, max(abs_bits(g.v[2 * j]), abs_bits(g.v[2 * j + 1])));
        }
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // values are v * 2^(own - 127); an e4m3 code is below 2^9
    const uint32_t own = X == F4_MX8 ? mx_byte : 127u;
    const uint32_t top = X == F4_MX8 ? own + 9 : (m >> 23) + 1;
    // 24: the eighth plane's scale stays above 2^-127 (smaller blocks keep 2^-125)
    g.byte = max(top, 24u);
    g.mul = __uint_as_float((127u + 22u + own - g.byte) << 23);
    g.twice = false;
    if (m >= 0x7F800000u || top > 254u) {
        // up to 2^128 after all, by the largest value there is (the smallest code is 2^-9)?
        const uint32_t most = own + max(m >> 23, 118u) - 126u;
        const bool good = m < 0x7F800000u && most <= 255u && own != 255u;
        g.twice = good && most == 255u;
        g.byte = good ? most - g.twice : 255u;
        g.mul = good ? __uint_as_float((127u + 22u + own - most) << 23) : 0.0f;
        if (!good) {
#pragma unroll
            for (int j = 0; j < 8; ++j) g.v[j] = 0.0f;
        }
    }
    return g;
}

// The e2m1 codes of the eight digits of eight values: word q holds plane q,
// the first value in the low bits.
QMM_DEVINL void f4_digits(const F4Group& g, uint32_t (&plane)[8]) {
    uint32_t a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // nearest integer to v * mul, |.| <= 2^22, plus 4 in every octal digit
        uint32_t u = __float_as_uint(fmaf(g.v[j], g.mul, 12582912.0f)) - 0x4B400000u + 0x00924924u;
        // octal digits to nibbles
        u += 15u * (u & 0x00FFF000u);
        u += 3u * (u & 0x0FC00FC0u);
        u += u & 0x38383838u;
        a[j] = u;
    }
    // transpose: 8 values x 8 nibbles
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        b[j] = prmt(a[j], a[j + 4], 0x5410);
        b[j + 4] = prmt(a[j], a[j + 4], 0x7632);
    }
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[j + i] = prmt(b[j + i], b[j + i + 2], 0x6240);
            a[j + i + 2] = prmt(b[j + i], b[j + i + 2], 0x7351);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const uint32_t M = 0x0F0F0F0Fu;
        b[j] = (a[j] & M) | ((a[j + 1] << 4) & ~M);
        b[j + 1] = ((a[j] >> 4) & M) | (a[j + 1] & ~M);
    }
    // digit d = u - 4 to the code of d / 2: the magnitude, plus 8 when negative
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const uint32_t u = b[7 - q];
        const uint32_t n = (~u >> 2) & 0x11111111u;
        plane[q] = ((u & 0x33333333u) ^ (3u * n)) + 9u * n;
    }
    if (g.twice) {  // codes 0 .. 4 of 0 .. 2 to those of 0 .. 4
        const uint32_t c = plane[0], M = 0x11111111u;
        plane[0] = c + (c & ~(c >> 1) & M) + 2u * (((c >> 1) | (c >> 2)) & M);
    }
}

// Scale bytes of plane q for four blocks from those of plane 0 (each at least
// 24; a NaN stays in plane 0, the others' codes are zero).
QMM_DEVINL uint32_t f4_plane_scale(uint32_t four, int q) { return four - 0x03030303u * (uint32_t)q; }

struct F4Params {
    MxTcParams c;
    const void* x;            // activations [x_rows, K] (values or e4m3 codes)
    const uint8_t* xs;        // their scale bytes when mxfp8
    const uint32_t* src;      // sorted row -> row, or null
    const int32_t* lhs;       // row -> x row, or null
    const int32_t* ids;       // grouped: expert of each y row
    int x_rows, E, cluster;
    int direct;               // grouped: every row is an item of its own
    int b_bytes;              // of a copy of planes
    uint32_t base, more;      // without items: tiles of a cluster, clusters with one more
    int k_base, k_more;       // k-blocks of a block, blocks of a cluster with one more
};

template <bool F16_, int X_, int BT_, int STAGES_>
struct MxF4 {
    static constexpr bool F16 = F16_;
    static constexpr int X = X_, BT = BT_, STAGES = STAGES_;
    static constexpr bool OWN = X != F4_PLANED;   // makes its planes itself
    static constexpr int NB = BT * F4_PLANES;     // columns: planes of a row beside one another
    static constexpr int SFB = (NB + 127) / 128;  // scale blocks of 128 columns
    static constexpr int A_BYTES = MT_ROWS * F4_BK / 2;
    static constexpr int B_BYTES = NB * F4_BK / 2;
    static constexpr int SG = 3;                  // ring of weight-scale groups (two k-blocks each)
    static constexpr int JOIN = BT <= 2 ? 7 : BT <= 16 ? 3 : 1;  // most other blocks of a cluster
    static constexpr int A_OFF = 0;
    static constexpr int B_OFF = A_OFF + STAGES * A_BYTES;
    static constexpr int SA_OFF = B_OFF + STAGES * B_BYTES;         // [SG][4][512]
    static constexpr int SB_OFF = SA_OFF + SG * 4 * 512;            // own planes: [STAGES][2][512]; else [SG][4][SFB * 512]
    static constexpr int SB_BYTES = OWN ? STAGES * 1024 : SG * 4 * SFB * 512;
    static constexpr int J_OFF = SB_OFF + SB_BYTES;                 // [JOIN][BT][128] floats
    static constexpr int BAR_OFF = J_OFF + JOIN * BT * MT_ROWS * 4;
    static constexpr int BARS = 3 * STAGES + 2 * SG + 4 + 8 + 1;
    static constexpr int SMEM = BAR_OFF + BARS * 8 + 32 + 1024;
    static constexpr int S_COLS = 2 * 4 * (1 + SFB);  // TMEM columns of a stage's scales
    static constexpr int ACCS = 2 * NB + STAGES * S_COLS <= 512 ? 2 : 1;
    static constexpr int USED = ACCS * NB + STAGES * S_COLS;
    static constexpr int COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
    static constexpr int THREADS = OWN ? 832 : 320;
    static_assert(USED <= 512, "tensor memory");
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(NB % 16 == 0 && NB <= 256 && (!OWN || BT <= 2), "MMA width");
};

// A cluster's tiles (a run, so that neighbours share an expert) and this
// block's k-blocks of each.
struct F4Walk {
    uint32_t tile, end;
    int k0, k1;
    QMM_DEVINL F4Walk(const F4Params& p, uint32_t rank) {
        uint32_t base = p.base, more = p.more, c, g;
        asm("mov.u32 %0, %%clusterid.x;" : "=r"(c));
        if (p.c.items) {  // their number is known here only
            asm("mov.u32 %0, %%nclusterid.x;" : "=r"(g));
            const uint32_t tiles = (uint32_t)p.c.n_tiles * (uint32_t)ld_dep(p.c.n_items);
            base = tiles / g;
            more = tiles - base * g;
        }
        tile = c * base + min(c, more);
        end = tile + base + (c < more);
        k0 = (int)rank * p.k_base + min((int)rank, p.k_more);
        k1 = k0 + p.k_base + ((int)rank < p.k_more);
    }
};

// The tiles of a run one after another.
struct F4Tiles {
    uint32_t tile, end;
    int item, nt;  // the tile is the nt-th of this item
    MxTile t;
    QMM_DEVINL F4Tiles(const F4Params& p, const F4Walk& w, int bt) : tile(w.tile), end(w.end) {
        item = tile < (uint32_t)p.c.n_tiles ? 0 : (int)(tile / (uint32_t)p.c.n_tiles);
        nt = (int)tile - item * p.c.n_tiles;
        if (more()) enter(p, bt);
    }
    QMM_DEVINL bool more() const { return tile < end; }
    QMM_DEVINL void enter(const F4Params& p, int bt) {
        t.row0 = item * bt;
        t.rows = min(bt, p.c.rows - t.row0);
        t.expert = 0;
        if (p.direct) {
            const uint32_t e = (uint32_t)ld_dep(p.ids + item);
            t.row0 = item;
            t.rows = e < (uint32_t)p.E ? 1 : 0;
            t.expert = t.rows ? (int)e : 0;
        } else if (p.c.items) {
            const int4 it = ld_dep(p.c.items + item);
            t.expert = it.x;
            t.row0 = it.y;
            t.rows = it.z;
        }
        t.n0 = nt * MT_ROWS;
    }
    // true when the next tile belongs to another item
    QMM_DEVINL bool next(const F4Params& p, int bt) {
        ++tile;
        t.n0 += MT_ROWS;
        if (++nt < p.c.n_tiles || !more()) return false;
        nt = 0;
        ++item;
        enter(p, bt);
        return true;
    }
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
    mx_f4_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_b,
                 const F4Params p) {
    using H = Half<C::F16>;
    constexpr int STAGES = C::STAGES, SG = C::SG;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bars = sbase + C::BAR_OFF;
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (STAGES + s); };
    auto digits = [&](int s) { return bars + 8 * (2 * STAGES + s); };
    auto scaled = [&](int g) { return bars + 8 * (3 * STAGES + g); };
    auto s_empty = [&](int g) { return bars + 8 * (3 * STAGES + SG + g); };
    auto acc_full = [&](int b) { return bars + 8 * (3 * STAGES + 2 * SG + b); };
    auto acc_empty = [&](int b) { return bars + 8 * (3 * STAGES + 2 * SG + 2 + b); };
    auto join_full = [&](int q) { return bars + 8 * (3 * STAGES + 2 * SG + 4 + q); };
    auto join_empty = [&](int q) { return bars + 8 * (3 * STAGES + 2 * SG + 8 + q); };
    const uint32_t started = bars + 8 * (3 * STAGES + 2 * SG + 12);  // the first activations are in
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + C::BARS * 8);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* reached = abort + 1;  // k-blocks the MMA warp has begun

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t S = (uint32_t)p.cluster, rank = mt_cluster_rank();
    if (threadIdx.x == 0) {
        *abort = 0;
        *reached = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(digits(s), C::BT);
        }
        for (int g = 0; g < SG; ++g) {
            mbar_init(scaled(g), 4);
            mbar_init(s_empty(g), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 4);
        }
        for (int q = 0; q < 4; ++q) {
            mbar_init(join_full(q), 1);
            mbar_init(join_empty(q), 1);
        }
        mbar_init(started, 1);
        mbar_fence_init();
        tma_prefetch_desc(&tmap_w);
        if constexpr (!C::OWN) tma_prefetch_desc(&tmap_b);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(C::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Barriers and tensor memory are ready after this; each role comes here once
    // its first lines are asked for (a load would hold the barrier up until its
    // data came).
    uint32_t tmem = 0;
    auto ready = [&]() {
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        // the other blocks' barriers are touched from the first join on
        if (S > 1) mt_cluster_arrive();
        tmem = *tmem_slot;
    };

    // With planes from a kernel before this one (a programmatic launch), the
    // other warps wait for it here and the TMA warp once the weights of its
    // first ring are on the way; without, the launch is an ordinary one.
    if (warp != 0 || p.c.items) pdl_wait();
    const F4Walk walk(p, rank);
    const int k0 = walk.k0, k1 = walk.k1;
    const int nk = k1 - k0, L = f4_ring_slots(C::OWN, nk, STAGES), fresh = f4_ring_fresh(C::OWN, nk, STAGES);

    if (warp == 0) {
        // ---------------- TMA ----------------
        auto load_w = [&](const MxTile& t, int kb, int s) {
            mbar_expect_tx(full(s), C::A_BYTES + (C::OWN ? 0 : (uint32_t)p.b_bytes));
            tma_load_2d(sbase + C::A_OFF + s * C::A_BYTES, &tmap_w, full(s), kb * (F4_BK / 2),
                        t.expert * p.c.N + t.n0);
        };
        F4Tiles tiles(p, walk, C::BT);
        ready();
        int i = 0, early = 0, s = 0;
        uint32_t ph = 0;
        if (!C::OWN && !p.c.items) {
            for (F4Tiles a = tiles; a.more() && early < STAGES; a.next(p, C::BT)) {
                for (int kb = k0; kb < k1 && early < STAGES; ++kb, ++early)
                    if (elect_one()) load_w(a.t, kb, early);
                __syncwarp();
            }
            pdl_wait();
        }
        for (; tiles.more() && !*abort; tiles.next(p, C::BT)) {
            const MxTile& t = tiles.t;
            for (int kb = k0; kb < k1; ++kb, ++i) {
                // The first activations and scales queue behind what weights are
                // already asked for; the rest of the ring follows them.
                if (C::OWN && i == F4_FIRST && !mt_wait(started, 0, abort, 1024)) break;
                if (!mt_wait(empty(s), ph ^ 1u, abort, 1)) break;
                if (elect_one()) {
                    if (i >= early) load_w(t, kb, s);
                    if constexpr (!C::OWN)
                        tma_load_2d(sbase + C::B_OFF + s * C::B_BYTES, &tmap_b, full(s), kb * (F4_BK / 2),
                                    t.row0 * F4_PLANES);
                }
                __syncwarp();
                if (++s == L) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- scale copies and MMAs ----------------
        ready();
        const uint32_t sf_cols = tmem + C::ACCS * C::NB;
        const uint64_t adesc0 = umma_desc_sw128(sbase + C::A_OFF), bdesc0 = umma_desc_sw128(sbase + C::B_OFF);
        int seg = 0, g = -1, s = 0, units = 0;  // tiles, scale groups so far; slot of the ring; k-blocks
        uint32_t ph = 0, made = 0;   // the slots' phases: all alike, and of the planes bit by bit
        int nt = (int)(walk.tile % (uint32_t)p.c.n_tiles), served = 0;  // place in the item; its tiles so far
        for (uint32_t tile = walk.tile; tile < walk.end && !*abort; ++tile) {
            const int b = seg % C::ACCS;
            const uint32_t acc = tmem + b * C::NB;
            if (!mt_wait(acc_empty(b), ((uint32_t)(seg / C::ACCS) & 1u) ^ 1u, abort, 2)) break;
            ++seg;
            for (int kb = k0; kb < k1; ++kb) {
                if (kb == k0 || (kb & 1) == 0) {
                    ++g;
                    if (!mt_wait(scaled(g % SG), (uint32_t)(g / SG) & 1u, abort, 8)) break;
                }
                if (C::OWN && served < fresh) {
                    if (!mt_wait(digits(s), (made >> s) & 1u, abort, 64)) break;
                    made ^= 1u << s;
                }
                if (!mt_wait(full(s), ph, abort, 4)) break;
                tc_fence_after();
                if (C::OWN && lane == 0) *reached = ++units;
                if (elect_one()) {
                    const uint32_t sfa = sf_cols + s * C::S_COLS, gs = (uint32_t)((g % SG) * 4 + (kb & 1) * 2);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // 128 k
                        const uint32_t col = sfa + h * 4 * (1 + C::SFB);
                        mt_copy_scales(col, sbase + C::SA_OFF + (gs + h) * 512);
#pragma unroll
                        for (int q = 0; q < C::SFB; ++q)
                            mt_copy_scales(col + 4 * (1 + q),
                                           sbase + C::SB_OFF +
                                               (C::OWN ? (s * 2 + h) * 512 : ((gs + h) * C::SFB + q) * 512));
                    }
                    const uint64_t ad = adesc0 + ((uint32_t)(s * C::A_BYTES) >> 4);
                    const uint64_t bd = bdesc0 + ((uint32_t)(s * C::B_BYTES) >> 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {  // 64 k: 32 bytes of a row
                        const uint32_t sf = sfa + (j >> 1) * 4 * (1 + C::SFB);
                        f4_mma(acc, ad + 2 * j, bd + 2 * j, f4_idesc(C::NB, (uint32_t)(j & 1) * 2), sf, sf + 4,
                               kb != k0 || j);
                    }
                    umma_commit(empty(s));
                    if ((kb & 1) || kb + 1 == k1) umma_commit(s_empty(g % SG));
                }
                __syncwarp();
                if (++s == L) {
                    s = 0;
                    ph ^= 1u;
                }
            }
            if (elect_one()) umma_commit(acc_full(b));
            __syncwarp();
            ++served;
            if (++nt == p.c.n_tiles) nt = served = 0;
        }
    } else if (warp < 6) {
        // ---------------- scales ----------------
        // Thread r owns row r of the weight tile and, with planes from a kernel
        // before, of each block of 128 columns.  A group is 16 bytes of a row
        // (512 k); loads run AHEAD groups ahead, across tiles.
        constexpr int NL = C::OWN ? 1 : 1 + C::SFB;
        constexpr int AHEAD = C::OWN ? 6 : 4;
        const int r = (warp - 2) * 32 + lane, n_sf = p.c.K / 32;
        const uint32_t at = sbase + (r & 31) * 16 + (r >> 5) * 4;
        const int g0 = k0 >> 1, g1 = (k1 - 1) >> 1;
        F4Tiles tiles(p, walk, C::BT);  // of the next load
        int grp = g0;
        const uint8_t* src[NL];
        auto rows_of = [&]() {
            const MxTile& t = tiles.t;
            src[0] = p.c.sfw + ((long long)t.expert * p.c.N + min(t.n0 + r, p.c.N - 1)) * n_sf;
#pragma unroll
            for (int q = 1; q < NL; ++q) {
                const int c = min((q - 1) * 128 + r, C::NB - 1);
                const long long row = min((long long)t.row0 * F4_PLANES + c, (long long)p.c.rows * F4_PLANES - 1);
                src[q] = p.c.sfb + row * p.c.sfb_row;
            }
        };
        auto load = [&](uint4 (&v)[NL]) {
            if (!tiles.more()) return;
            if (p.c.vec_w == 16) {
                v[0] = ldg_v4(src[0] + 16 * grp);
#pragma unroll
                for (int q = 1; q < NL; ++q) v[q] = ld_v4(src[q] + 16 * grp);
            } else {
                v[0] = mt_scale_bytes(src[0], 16 * grp, n_sf, p.c.vec_w, p.c.sfw, p.c.sfw_end);
#pragma unroll
                for (int q = 1; q < NL; ++q) v[q] = ld_v4(src[q] + 16 * grp);
            }
            if (++grp > g1) {
                grp = g0;
                tiles.next(p, C::BT);
                rows_of();
            }
        };
        uint4 v[AHEAD][NL];
        if (tiles.more()) {
            rows_of();
#pragma unroll
            for (int q = 0; q < NL; ++q) mt_prefetch(src[q] + 16 * grp);
        }
        ready();
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) load(v[a]);
        const int total = (int)(walk.end - walk.tile) * (g1 - g0 + 1);
        for (int base = 0; base < total && !*abort; base += AHEAD) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int g = base + a;
                if (g >= total) break;
                if (!mt_wait(s_empty(g % SG), ((uint32_t)(g / SG) & 1u) ^ 1u, abort, 16)) break;
                const uint32_t slot = (uint32_t)(g % SG) * 4;
#pragma unroll
                for (int q = 0; q < NL; ++q) {
                    const uint32_t w[4] = {v[a][q].x, v[a][q].y, v[a][q].z, v[a][q].w};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t to = q ? C::SB_OFF + ((slot + c) * C::SFB + q - 1) * 512
                                              : C::SA_OFF + (slot + c) * 512;
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + to), "r"(w[c]) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(scaled(g % SG));
                load(v[a]);
            }
        }
    } else if (warp < 10) {
        // ---------------- epilogue ----------------
        ready();
        const int quarter = warp & 3, row = quarter * 32 + lane;  // weight row of the tile = TMEM lane
        const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
        if (p.ids)  // y rows whose id has no expert
            for (int r = blockIdx.x * 4 + warp - 6; r < p.c.rows; r += gridDim.x * 4)
                if ((uint32_t)ld_dep(p.ids + r) >= (uint32_t)p.E)
                    for (int n = lane; n < p.c.N; n += 32) p.c.y[(long long)r * p.c.N + n] = 0;
        if (S > 1) mt_cluster_wait();
        // a block's sums: [rows / PER][128 weight rows][PER]
        constexpr int PER = C::BT < 4 ? C::BT : 4;  // rows of a TMEM load
        const uint32_t j_row = sbase + C::J_OFF + row * (PER * 4);
        const uint32_t to = S > 1 && rank ? mt_remote(j_row + (rank - 1) * (C::BT * MT_ROWS * 4), 0) : 0;
        const uint32_t to_full = S > 1 && rank ? mt_remote(join_full(quarter), 0) : 0;
        int seg = 0;
        for (F4Tiles tiles(p, walk, C::BT); tiles.more() && !*abort; tiles.next(p, C::BT)) {
            const MxTile& t = tiles.t;
            int out_l = t.row0 + lane;  // y row of row `lane`
            if (p.c.dst && lane < t.rows) out_l = (int)ld_dep(p.c.dst + t.row0 + lane);
            const int b = seg % C::ACCS;
            const uint32_t j_ph = (uint32_t)seg & 1u;
            if (S > 1 && rank == 0 && lane == 0)  // the other blocks' sums of these 32 weight rows
                mbar_expect_tx(join_full(quarter), (S - 1) * (uint32_t)((t.rows + PER - 1) / PER * PER) * 128);
            if (!mt_wait(acc_full(b), (uint32_t)(seg / C::ACCS) & 1u, abort, 32)) break;
            if (S > 1) {
                if (rank ? !mt_wait(join_empty(quarter), j_ph ^ 1u, abort, 128)
                         : !mt_wait<true>(join_full(quarter), j_ph, abort, 256))
                    break;
            }
            ++seg;
            tc_fence_after();
            const int n = t.n0 + row;
#pragma unroll 1
            for (int j0 = 0; j0 < t.rows; j0 += PER) {
                uint32_t u[PER * 8];
                if constexpr (PER == 4) tmem_ld32(t_lane + b * C::NB + j0 * F4_PLANES, u);
                else tmem_ld16(t_lane + b * C::NB + j0 * F4_PLANES, u);
                tmem_wait_ld();
                float f[PER];
#pragma unroll
                for (int d = 0; d < PER; ++d) {
                    f[d] = __uint_as_float(u[8 * d + 7]);  // small to large
#pragma unroll
                    for (int q = 6; q >= 0; --q) f[d] += __uint_as_float(u[8 * d + q]);
                }
                if (rank != 0) {
                    mt_remote_store(to + j0 * (MT_ROWS * 4), f, to_full);
                    continue;
                }
                for (uint32_t o = 0; o + 1 < S; ++o) {
                    const uint32_t from = j_row + (o * C::BT + j0) * (MT_ROWS * 4);
                    float part[4] = {};
                    if constexpr (PER == 4)
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(part[0]), "=f"(part[1]), "=f"(part[2]), "=f"(part[3])
                                     : "r"(from)
                                     : "memory");
                    else
                        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                                     : "=f"(part[0]), "=f"(part[1])
                                     : "r"(from)
                                     : "memory");
#pragma unroll
                    for (int d = 0; d < PER; ++d) f[d] += part[d];
                }
#pragma unroll
                for (int d = 0; d < PER; ++d) {
                    const long long out = __shfl_sync(0xffffffffu, out_l, (j0 + d) & 31);
                    if (j0 + d < t.rows && n < p.c.N) p.c.y[out * p.c.N + n] = H::from_f32(f[d]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(acc_empty(b));
                if (rank == 0 && tiles.tile + 1 < tiles.end)
                    for (uint32_t o = 1; o < S; ++o) mt_pair_arrive(mt_remote(join_empty(quarter), o));
            }
        }
    } else if constexpr (C::OWN) {
        // ---------------- activations to digits ----------------
        // A warp takes one row of one k-block: lane l the values 8l .. 8l + 7.
        // The 16 warps divide a tile's rows, and with fewer rows the k-blocks
        // too: of `par` sets of warps each takes every par-th k-block of the run
        // of tiles.  Loads run AHEAD of a warp's k-blocks ahead, across tiles.
        constexpr int AHEAD = 2;
        const int w = warp - 10, n_sf = p.c.K / 32;
        struct Step {
            uint4 raw;
            uint32_t byte;
            int i;         // k-block of the run, -1 past the end
            int tok, fill; // row; arrivals this warp owes (the first row's warp for the rows a tile lacks)
            bool live;
        } st[AHEAD];
        F4Tiles tiles(p, walk, C::BT);  // of the next load
        int i0 = 0, kb = 0, par = 1, part = 0, tok = 0, rows = 0, served = 0;
        const char* xrow = nullptr;
        const uint8_t* srow = nullptr;
        auto row_of = [&]() {
            const MxTile& t = tiles.t;
            rows = max(t.rows, 1);
            par = min(16 / rows, L);
            part = w / rows;
            tok = w - part * rows;
            xrow = nullptr;
            if (part >= par || t.rows == 0) return;
            long long xr = t.row0 + tok;
            if (p.src) xr = ld_dep(p.src + xr);
            if (p.lhs) xr = (uint32_t)ld_dep(p.lhs + xr);
            xr = xr < p.x_rows ? xr : p.x_rows - 1;
            xrow = static_cast<const char*>(p.x) + xr * (p.c.K * (C::X == F4_MX8 ? 1LL : 2LL));
            if constexpr (C::X == F4_MX8) srow = p.xs + xr * n_sf;
        };
        auto step = [&]() {  // to the next tile that needs planes
            i0 += nk;
            ++served;
            bool other = tiles.next(p, C::BT);
            if (!other && served == fresh && tiles.more()) {
                // the item's last tile of this run, then the one after it
                const int skip = min(p.c.n_tiles - tiles.nt, (int)(tiles.end - tiles.tile)) - 1;
                tiles.tile += skip;
                tiles.nt += skip;
                i0 += (skip + 1) * nk;
                other = tiles.next(p, C::BT);
            }
            if (other) {
                served = 0;
                row_of();
            }
        };
        auto enter = [&]() {  // this warp's first k-block in the tile or a later one
            while (tiles.more()) {
                int d = part - i0 % par;
                if (d < 0) d += par;
                kb = k0 + d;
                if (part < par && kb < k1) return;
                step();
            }
        };
        auto load = [&](Step& s) {
            s.i = -1;
            if (!tiles.more()) return;
            s.raw = make_uint4(0, 0, 0, 0);
            s.byte = 127;
            s.i = i0 + kb - k0;
            s.tok = tok;
            s.fill = tok ? 1 : C::BT - rows + 1;
            s.live = xrow != nullptr;
            const int k = kb * F4_BK + lane * 8;
            if (s.live && k < p.c.K) {
                if constexpr (C::X == F4_MX8) {
                    const uint2 q = ld_dep(reinterpret_cast<const uint2*>(xrow + k));
                    s.raw.x = q.x;
                    s.raw.y = q.y;
                    s.byte = ld_dep(srow + (k >> 5));
                } else {
                    s.raw = ld_v4(xrow + 2 * k);
                }
            }
            kb += par;
            if (kb >= k1) {
                step();
                enter();
            }
        };
        if (tiles.more()) {
            row_of();
            const int k = min((k0 + part) * F4_BK + lane * 8, p.c.K - 8);
            if (xrow) mt_prefetch(xrow + (C::X == F4_MX8 ? k : 2 * k));
        }
        ready();
        enter();
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) load(st[a]);
        int seen = -1;  // last k-block whose slot this warp waited for
#pragma unroll 1
        while (st[0].i >= 0 && !*abort) {
            const int i = st[0].i, turn = i / L, s = i - turn * L;
            uint32_t plane[8], four = 0;
            if (st[0].live) {
                const F4Group g = f4_group<C::X>(st[0].raw, st[0].byte);
                f4_digits(g, plane);
                // this half-warp's four blocks: scale bytes as one word
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    four |= __shfl_sync(0xffffffffu, g.byte, (lane & 16) + 4 * c) << (8 * c);
                if (const uint32_t twice = __ballot_sync(0xffffffffu, g.twice)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        four += (lane & 15) ? ((twice >> ((lane & 16) + 4 * c)) & 1u) << (8 * c) : 0u;
                }
            }
            // a warp that had nothing to do for more than a ring first lets the
            // MMA warp come within one (which it can without this warp)
            bool gone = false;
            if (i - seen > L) {
                int tries = 0;
                while (!f4_ring_may_wait(*reached, i, L) && !*abort) {
                    __nanosleep(100);
                    if (++tries < (1 << 20)) continue;
                    *abort = 1;
                    atomicCAS(&g_mx_error, 0, 2048);
                }
                gone = __any_sync(0xffffffffu, *abort);
            }
            if (gone || !mt_wait(empty(s), ((uint32_t)turn & 1u) ^ 1u, abort, 512)) break;
            seen = i;
            if (st[0].live) {
                const uint32_t b =
                    sbase + C::B_OFF + s * C::B_BYTES + st[0].tok * F4_PLANES * 128 + (lane & 3) * 4;
#pragma unroll
                for (int q = 0; q < 8; ++q)  // 128-byte swizzle: chunk ^ row
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(b + q * 128 + (((lane >> 2) ^ q) << 4)),
                                 "r"(plane[q])
                                 : "memory");
                const int q = lane & 15, c = st[0].tok * F4_PLANES + q;
                if (q < 8)
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(sbase + C::SB_OFF + (s * 2 + (lane >> 4)) * 512 +
                                                                 (c & 31) * 16 + (c >> 5) * 4),
                                 "r"(f4_plane_scale(four, q))
                                 : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(digits(s)), "r"(st[0].fill)
                             : "memory");
            if (i == 0 && st[0].tok == 0 && lane == 0) mbar_arrive(started);
#pragma unroll
            for (int a = 0; a + 1 < AHEAD; ++a) st[a] = st[a + 1];
            load(st[AHEAD - 1]);
        }
    }
    if (*abort) __nanosleep(1000000);  // after a wait gave up: let copies in flight land
    if (S > 1) {
        // every thread arrives twice and waits twice; a block's shared memory
        // outlives the others' last access to it
        __syncwarp();
        if (warp < 6 || warp >= 10) mt_cluster_wait();
        __syncwarp();
        mt_cluster_arrive();
        mt_cluster_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
    }
}

// The planes, where another kernel makes them: [R][8][K/2] with scales [R][8][K/32
// rounded up to 16], rows taken through src and lhs; four lanes hold a block.
template <int X>
__global__ void __launch_bounds__(64) mx_f4_planes_kernel(const void* x, const uint8_t* xs, uint32_t* planes,
                                                           uint8_t* scales, const uint32_t* src, const int32_t* lhs,
                                                           int x_rows, int R, int K) {
    pdl_launch_dependents();
    const int n8 = K / 8, pitch = (K / 32 + 15) & ~15;
    const long long total = (long long)R * n8, step = (long long)gridDim.x * blockDim.x;
    for (long long base = ((long long)blockIdx.x * blockDim.x + threadIdx.x) & ~31LL; base < total; base += step) {
        const long long i = base + (threadIdx.x & 31);
        const bool in = i < total;
        const int r = in ? (int)(i / n8) : 0, c = (int)(i - (long long)r * n8);
        uint4 raw = make_uint4(0, 0, 0, 0);
        uint32_t byte = 127;
        if (in) {
            long long xr = r;
            if (src) xr = ld_dep(src + xr);
            if (lhs) xr = (uint32_t)ld_dep(lhs + xr);
            xr = xr < x_rows ? xr : x_rows - 1;
            if constexpr (X == F4_MX8) {
                const uint2 q = ld_dep(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(x) + xr * K) + c);
                raw.x = q.x;
                raw.y = q.y;
                byte = ld_dep(xs + xr * (K / 32) + (c >> 2));
            } else {
                raw = ld_v4(static_cast<const uint16_t*>(x) + xr * K + c * 8);
            }
        }
        const F4Group g = f4_group<X>(raw, byte);
        uint32_t plane[8];
        f4_digits(g, plane);
        if (!in) continue;
        uint32_t* to = planes + (long long)r * F4_PLANES * n8 + c;
        uint8_t* sf = scales + (long long)r * F4_PLANES * pitch + (c >> 2);
#pragma unroll
        for (int q = 0; q < F4_PLANES; ++q) {
            to[q * n8] = plane[q];
            if ((c & 3) == 0) sf[q * pitch] = (uint8_t)(f4_plane_scale(g.byte, q) + (q ? g.twice : 0));
        }
        if (c + 4 == n8 && n8 < 4 * pitch) {  // the last block's first lane: the rest of the rows
#pragma unroll 1
            for (int q = 0; q < F4_PLANES; ++q)
#pragma unroll 1
                for (int k = 1; k <= pitch - n8 / 4; ++k) sf[q * pitch + k] = 0;
        }
    }
}

}  // namespace qmm

namespace qmm_host {

namespace {

long long f4_items_max(long long rows, long long E, int bt, bool grouped) {
    return grouped ? rows / bt + (E < rows ? E : rows) + 1 : (rows + bt - 1) / bt;
}

// Most clusters of S blocks that run at once (one block on an SM).
template <class C>
int f4_clusters(int S, cudaLaunchConfig_t& cfg) {
    static int known[9] = {};
    if (known[S]) return known[S];
    int n = 0;
    cfg.gridDim = dim3((unsigned)(S * (kMxMaxBlocks / S)));
    if (cudaOccupancyMaxActiveClusters(&n, qmm::mx_f4_kernel<C>, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = mx_sm_count() / S / 2;
    }
    known[S] = n < 1 ? 1 : n;
    return known[S];
}

// Blocks of a cluster: k-blocks one after another on a block cost about 0.23 us
// (what an SM takes in), all of them together 2.7 ns (HBM), and a join about
// as much as two k-blocks.
template <class C>
int launch_f4(const MxMatmul& a, const CUtensorMap& mw, const CUtensorMap& mb, qmm::F4Params& p, double tiles) {
    auto kern = qmm::mx_f4_kernel<C>;
    int rc = ensure_smem_limit((const void*)kern, C::SMEM, "mx_f4 smem attribute");
    if (rc) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = a.st;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    int best = 1, clusters = 1;
    double least = 0;
    for (int S = 1; S <= C::JOIN + 1 && S <= p.c.KB; ++S) {
        at[0].val.clusterDim.x = (unsigned)S;
        cfg.numAttrs = 1;
        int n = f4_clusters<C>(S, cfg);
        if (n > tiles) n = tiles < 1 ? 1 : (int)tiles;
        const double rounds = (double)(long long)((tiles + n - 1) / n);
        const double own = rounds * ((p.c.KB + S - 1) / S) * 0.23, all = tiles * p.c.KB * 0.0027;
        const double us = (own > all ? own : all) + (S > 1 ? 0.5 : 0.0);
        if (S == 1 || us < least) {
            least = us;
            best = S;
            clusters = n;
        }
    }
    p.cluster = best;
    const unsigned whole = (unsigned)tiles;
    p.base = whole / (unsigned)clusters;
    p.more = whole % (unsigned)clusters;
    p.k_base = p.c.KB / best;
    p.k_more = p.c.KB % best;
    at[0].val.clusterDim.x = (unsigned)best;
    cfg.gridDim = dim3((unsigned)(best * clusters));
    cfg.numAttrs = !C::OWN && pdl_enabled() ? 2 : 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kern, mw, mb, p), "mx_f4 launch");
}

template <bool F16, int X>
int launch_f4_bt(const MxMatmul& a, const CUtensorMap& mw, const CUtensorMap& mb, qmm::F4Params& p, double tiles,
                 int bt) {
    using namespace qmm;
    if (bt == 2) return launch_f4<MxF4<F16, X, 2, 10>>(a, mw, mb, p, tiles);
    if (bt == 16) return launch_f4<MxF4<F16, F4_PLANED, 16, 5>>(a, mw, mb, p, tiles);
    return launch_f4<MxF4<F16, F4_PLANED, 32, 3>>(a, mw, mb, p, tiles);
}

}  // namespace

// A few rows over many experts: hardly any two meet, so each is an item of its
// own and nothing is sorted.
bool mx_f4_direct(long long rows, long long E, bool grouped) { return grouped && rows <= 32 && 4 * rows <= E; }

// Rows of a tile, 0 where the kernel is not for this size.
int mx_f4_item_rows(long long rows, long long E, long long N, long long K, bool mx, bool grouped) {
    const long long mean = (rows + E - 1) / E;
    // The kernel of mx_tc.cu spreads the weights' codes, but multiplies by one to
    // three planes where this one has the rate of four of them: it is ahead
    // from few rows on for mxfp8 and later for 16-bit activations, later still
    // where its larger tiles are few.  Here / there, us: mxfp8 16 rows of
    // 17408x5120 14.7 / 18.9, 64 rows 27.1 / 20.0, 64 of 1024x5120 12.8 / 10.7;
    // bf16 64 rows of 17408x5120 27.1 / 27.2, 96 rows 36.6 / 28.8, 96 of
    // 6144x5120 16.4 / 21.5, 128 of it 25.2 / 24.0; 32 experts of 1024x2048 with
    // 24 rows each 24.3 / 28.8 (mxfp8 24.5 / 23.3), with 32 rows 31.2 / 29.9.
    if (mx ? mean > 16
           : grouped ? mean > 24 : mean > 64 && (mean + 31) / 32 * ((N + 127) / 128) > kMxMaxBlocks)
        return 0;
    if (mx_f4_direct(rows, E, grouped)) return 2;
    // One launch for a product that is about as short as a launch; with planes
    // made by a kernel before it the weight stream itself is faster (one row of
    // 1024x5120: 6.7 us against 6.9, of 17408x5120: 14.2 against 13.2).
    if (!grouped && rows <= 2 && N * K <= 1LL << 24) return 2;
    // An expert's rows beyond one tile read its weights again: room for twice
    // the mean.
    return (grouped ? 2 * mean : mean) <= 16 ? 16 : 32;
}

bool mx_f4_takes(long long rows, long long E, long long N, long long K, bool mx, bool grouped) {
    const int bt = mx_f4_item_rows(rows, E, N, K, mx, grouped);
    return bt && E * N <= (1LL << 31) - 256 && rows * qmm::F4_PLANES <= (1LL << 31) - 256 &&
           f4_items_max(rows, E, bt, true) * ((N + 127) / 128) * ((K + 255) / 256) < (1LL << 31);
}

size_t mx_f4_workspace(long long rows, long long K, int bt) {
    return bt == 2 ? 0
                   : mx_al256((size_t)qmm::F4_PLANES * rows * (K / 2)) +
                         mx_al256((size_t)qmm::F4_PLANES * rows * mx_plane_row(K));
}

int launch_mx_f4(const MxMatmul& a, const int4* items, const int32_t* n_items, const int32_t* ids, int bt, void* ws) {
    const bool grouped = ids != nullptr, own = bt == 2;
    uint32_t* planes = static_cast<uint32_t*>(ws);
    uint8_t* scales = static_cast<uint8_t*>(ws) + mx_al256((size_t)qmm::F4_PLANES * a.rows * (a.K / 2));
    qmm::F4Params p{};
    p.c.sfw = a.ws;
    p.c.sfb = own ? nullptr : scales;
    p.c.y = static_cast<uint16_t*>(a.y);
    p.c.items = items;
    p.c.n_items = n_items;
    p.c.dst = a.dst;
    p.c.rows = (int)a.rows;
    p.c.N = (int)a.N;
    p.c.K = (int)a.K;
    p.c.KB = (int)((a.K + qmm::F4_BK - 1) / qmm::F4_BK);
    p.c.n_tiles = (int)((a.N + 127) / 128);
    p.c.sfw_end = a.ws + a.E * a.N * (a.K / 32);
    p.c.sfb_row = (int)mx_plane_row(a.K);
    p.c.vec_w = mx_scale_vec(a.K, a.ws);
    p.x = a.x;
    p.xs = a.xs;
    p.src = a.src;
    p.lhs = a.lhs;
    p.ids = ids;
    p.x_rows = (int)a.x_rows;
    p.E = (int)a.E;
    p.direct = grouped && !items;
    // grouped: how many tiles there are is known on the device; estimate from
    // evenly spread rows
    double n = (double)f4_items_max(a.rows, a.E, bt, false);
    if (p.direct) n = (double)a.rows;
    else if (grouped) {
        // share of experts without a row: (1 - 1/E)^rows
        const double miss = a.E > 1 ? std::exp((double)a.rows * std::log1p(-1.0 / (double)a.E)) : 0.0;
        n += (1.0 - miss) * (double)a.E;
        if (n > (double)a.rows) n = (double)a.rows;
    }
    CUtensorMap mw, mb;
    const uint64_t row = (uint64_t)a.K / 2;
    int rc = tensor_map_2d(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, row, (uint64_t)(a.E * a.N), row, 128, 128,
                           CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    mb = mw;
    if (!own) {
        // no taller than the batch: a copy mostly out of range is slower (5 rows of
        // 17408x5120: 16.7 us with a box for 16, 15.0 with one for 5)
        const int box = (int)(a.rows < bt ? a.rows : bt) * qmm::F4_PLANES;
        p.b_bytes = box * (qmm::F4_BK / 2);
        rc = tensor_map_2d(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, planes, row, (uint64_t)a.rows * qmm::F4_PLANES, row,
                           128, (uint32_t)box, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc) return rc;
        const long long want = (a.rows * (a.K / 8) + 63) / 64;
        const unsigned g = (unsigned)(want < 148 * 32 ? want : 148 * 32);
#define QMM_PLANES(X)                                                                                                \
    qmm::mx_f4_planes_kernel<X><<<g, 64, 0, a.st>>>(a.x, a.xs, planes, scales, a.src, a.lhs, (int)a.x_rows,          \
                                                     (int)a.rows, (int)a.K)
        if (a.xs) QMM_PLANES(qmm::F4_MX8);
        else if (a.f16) QMM_PLANES(qmm::F4_FP16);
        else QMM_PLANES(qmm::F4_BF16);
#undef QMM_PLANES
        rc = cuda_status(cudaGetLastError(), "mx_f4_planes launch");
        if (rc) return rc;
    }
    const double tiles = n * p.c.n_tiles;
    if (a.xs) return a.f16 ? launch_f4_bt<true, qmm::F4_MX8>(a, mw, mb, p, tiles, bt)
                           : launch_f4_bt<false, qmm::F4_MX8>(a, mw, mb, p, tiles, bt);
    return a.f16 ? launch_f4_bt<true, qmm::F4_FP16>(a, mw, mb, p, tiles, bt)
                 : launch_f4_bt<false, qmm::F4_BF16>(a, mw, mb, p, tiles, bt);
}

int mx_f4_device_error(int reset) { return mx_error_flag(reset); }

}  // namespace qmm_host
