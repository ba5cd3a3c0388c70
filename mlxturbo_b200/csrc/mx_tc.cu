// mx_tc.cu -- products with mxfp4 weights on the block-scaled tensor-core
// instructions (tcgen05.mma kind::mxf8f6f4), dense and grouped by expert.
//
//   y[m, n] = sum_k w[n, k] * x[m, k],   w = e2m1 code * 2^e per 32 values
//
// The weights are the A operand exactly as stored: TMA spreads 16 packed codes
// over 16 bytes of shared memory on the way in, the instruction multiplies the
// codes and applies one scale byte per row and 32 values itself, so no thread
// ever touches a weight.  The B operand is e4m3.  mxfp8 activations are that
// already.  A 16-bit activation is the sum of P e4m3 planes, each with its own
// block scale (mx_planes_kernel):
//
//   x = 2^e0 c0 + 2^(e0-4) c1 (+ 2^(e0-8) c2),  e0 = floor(log2 max|block|) - 7
//
// A code holds four significant bits and the remainder of rounding to nearest
// has one bit less than the half unit it is bounded by, so two planes hold the
// 8 significant bits of bf16 and three the 11 of fp16, exactly, for values down
// to 2^-14 of the largest in their block of 32; below that the smallest code of
// the last plane leaves 2^-21 (bf16) or 2^-25 (fp16) of that largest value.
// Products and sums are fp32 in TMEM.
//
// One block computes 128 weight rows x BT activation rows:
//   warp 0      TMA: weights and planes into a ring of STAGES k-blocks of 128
//   warp 1      tensor memory, scale copies (tcgen05.cp) and the MMAs
//   warps 2..5  scale bytes into the instruction's layout in shared memory
//   warps 6..9  epilogue: TMEM -> y, or a partial sum
// Blocks are persistent.  Work is counted in k-blocks of tiles.  With enough
// tiles each block takes whole ones; with few, the k-blocks are divided evenly
// over the blocks, a tile shared by several is joined by the last of them to
// finish, in the order of k, so results do not depend on timing.

#include "mx_mma.cuh"

namespace qmm {

constexpr int MT_BK = 128;    // K of a stage

QMM_DEVINL void mt_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// Instruction descriptor: A e2m1 (5), B e4m3 (0), both K-major, ue8m0 scales,
// scale byte `id` of the four in a TMEM column for both operands.
QMM_DEVINL constexpr uint32_t mt_idesc(int N, uint32_t id) {
    return (id << 4) | (5u << 7) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(MT_ROWS >> 7) << 27) |
           (id << 29);
}

// PCOL: the planes are columns of one MMA (BT * P wide; weights cross shared
// memory once); else they are further K of the same accumulator.
template <bool F16_, int P_, bool PCOL_, int BT_, int STAGES_>
struct MxTc {
    static constexpr bool F16 = F16_, PCOL = PCOL_;
    static constexpr int P = P_, BT = BT_, STAGES = STAGES_;
    static constexpr int NB = PCOL ? P * BT : BT;  // columns of one MMA
    static constexpr int PK = PCOL ? 1 : P;
    static constexpr int SFB = (NB + 127) / 128;   // scale blocks of a plane
    static constexpr int A_BYTES = MT_ROWS * MT_BK;
    static constexpr int A_TX = A_BYTES / 2;  // what a copy of packed codes counts on its barrier: the codes
    static constexpr int B_BYTES = PK * NB * MT_BK;
    static constexpr int S_BYTES = 512 * (1 + PK * SFB);  // scales of a k-block
    static constexpr int SG = 3;                          // ring of scale groups (four k-blocks each)
    static constexpr int A_OFF = 0;
    static constexpr int B_OFF = A_OFF + STAGES * A_BYTES;
    static constexpr int S_OFF = B_OFF + STAGES * B_BYTES;
    static constexpr int BAR_OFF = S_OFF + SG * 4 * S_BYTES;
    static constexpr int BARS = 2 * STAGES + 2 * SG + 4;
    static constexpr int SMEM = BAR_OFF + BARS * 8 + 32 + 1024;
    static constexpr int S_COLS = 4 * (1 + PK * SFB);  // TMEM columns of a stage's scales
    static constexpr int ACCS = 2 * NB + STAGES * S_COLS <= 512 ? 2 : 1;
    static constexpr int USED = ACCS * NB + STAGES * S_COLS;
    static constexpr int COLS = USED <= 32 ? 32 : USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
    static constexpr int THREADS = 320;
    static_assert(USED <= 512, "tensor memory");
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(NB % 16 == 0 && NB <= 256 && BT % 8 == 0, "MMA width");
};

template <int CH>
QMM_DEVINL void mt_tmem_ld(uint32_t taddr, uint32_t (&v)[CH]) {
    if constexpr (CH == 8) tmem_ld8(taddr, v);
    else tmem_ld16(taddr, v);
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
    mx_tc_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_b,
                 const MxTcParams p) {
    using H = Half<C::F16>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bars = sbase + C::BAR_OFF;
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (STAGES + s); };
    auto scaled = [&](int g) { return bars + 8 * (2 * STAGES + g); };
    auto s_empty = [&](int g) { return bars + 8 * (2 * STAGES + C::SG + g); };
    auto acc_full = [&](int b) { return bars + 8 * (2 * STAGES + 2 * C::SG + b); };
    auto acc_empty = [&](int b) { return bars + 8 * (2 * STAGES + 2 * C::SG + 2 + b); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + C::BARS * 8);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        *abort = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int g = 0; g < C::SG; ++g) {
            mbar_init(scaled(g), 4);
            mbar_init(s_empty(g), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 4);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tmap_w);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(C::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t sf_cols = tmem + C::ACCS * C::NB;

    // Everything but the weights of a dense call may come from the kernel
    // before this one, so the other warps wait for it here, and the TMA warp
    // once the weights of its first ring are on the way.
    if (warp != 0 || p.items) pdl_wait();
    const uint32_t tiles =
        (uint32_t)p.n_tiles * (uint32_t)(p.items ? ld_dep(p.n_items) : (p.rows + C::BT - 1) / C::BT);
    MxWalk walk(p, tiles);
    uint32_t tile;
    int k0, k1;

    if (warp == 0) {
        // ---------------- TMA ----------------
        auto load_w = [&](const MxTile& t, int kb, int s) {
            mbar_expect_tx(full(s), C::A_TX + C::B_BYTES);
            tma_load_2d(sbase + C::A_OFF + s * C::A_BYTES, &tmap_w, full(s), kb * MT_BK, t.expert * p.N + t.n0);
        };
        auto load_b = [&](const MxTile& t, int kb, int s) {
#pragma unroll
            for (int q = 0; q < C::P; ++q)
                tma_load_2d(sbase + C::B_OFF + s * C::B_BYTES + q * C::BT * MT_BK, &tmap_b, full(s), kb * MT_BK,
                            q * p.rows + t.row0);
        };
        int i = 0, early = 0;
        if (!p.items) {
            MxWalk ahead = walk;
            while (early < STAGES && ahead.next(tile, k0, k1)) {
                const MxTile t = mt_tile(p, tile, C::BT);
                for (int kb = k0; kb < k1 && early < STAGES; ++kb, ++early)
                    if (elect_one()) load_w(t, kb, early);
                __syncwarp();
            }
            pdl_wait();
        }
        while (walk.next(tile, k0, k1) && !*abort) {
            const MxTile t = mt_tile(p, tile, C::BT);
            for (int kb = k0; kb < k1; ++kb, ++i) {
                const int s = i % STAGES;
                if (!mt_wait(empty(s), ((uint32_t)(i / STAGES) & 1u) ^ 1u, abort, 1)) break;
                if (elect_one()) {
                    if (i >= early) load_w(t, kb, s);
                    load_b(t, kb, s);
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ---------------- scale copies and MMAs ----------------
        const uint64_t adesc0 = umma_desc_sw128(sbase + C::A_OFF), bdesc0 = umma_desc_sw128(sbase + C::B_OFF);
        int i = 0, seg = 0, g = -1;  // k-blocks, stretches and scale groups so far
        while (walk.next(tile, k0, k1) && !*abort) {
            const int b = seg % C::ACCS;
            const uint32_t acc = tmem + b * C::NB;
            if (!mt_wait(acc_empty(b), ((uint32_t)(seg / C::ACCS) & 1u) ^ 1u, abort, 2)) break;
            ++seg;
            for (int kb = k0; kb < k1; ++kb, ++i) {
                const int s = i % STAGES;
                if (kb == k0 || (kb & 3) == 0) {
                    ++g;
                    if (!mt_wait(scaled(g % C::SG), (uint32_t)(g / C::SG) & 1u, abort, 8)) break;
                }
                if (!mt_wait(full(s), (uint32_t)(i / STAGES) & 1u, abort, 4)) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t sfa = sf_cols + s * C::S_COLS;
                    const uint32_t ssm = sbase + C::S_OFF + ((g % C::SG) * 4 + (kb & 3)) * C::S_BYTES;
#pragma unroll
                    for (int q = 0; q < 1 + C::PK * C::SFB; ++q) mt_copy_scales(sfa + 4 * q, ssm + 512 * q);
                    const uint64_t ad = adesc0 + ((uint32_t)(s * C::A_BYTES) >> 4);
                    const uint64_t bd = bdesc0 + ((uint32_t)(s * C::B_BYTES) >> 4);
#pragma unroll
                    for (int q = 0; q < C::PK; ++q)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mt_mma(acc, ad + 2 * j, bd + ((q * C::NB * MT_BK) >> 4) + 2 * j,
                                   mt_idesc(C::NB, (uint32_t)j), sfa, sfa + 4 * (1 + q * C::SFB),
                                   kb != k0 || q || j);
                    umma_commit(empty(s));
                    if ((kb & 3) == 3 || kb + 1 == k1) umma_commit(s_empty(g % C::SG));
                }
                __syncwarp();
            }
            if (elect_one()) umma_commit(acc_full(b));
            __syncwarp();
        }
    } else if (warp < 6) {
        // ---------------- scales ----------------
        // Thread r owns row r of the weight tile and of each block of 128 MMA
        // columns; a row's words of four k-blocks are one 16-byte load where
        // rows are that aligned.  Loads run three groups ahead.
        constexpr int NL = 1 + C::PK * C::SFB;
        constexpr int AHEAD = 3;
        const int r = (warp - 2) * 32 + lane;
        const uint32_t sdst = sbase + C::S_OFF + (r & 31) * 16 + (r >> 5) * 4;
        int g = 0;
        while (walk.next(tile, k0, k1) && !*abort) {
            const MxTile t = mt_tile(p, tile, C::BT);
            const uint8_t* src[NL];
            const int n_sf = p.KB * 4;
            src[0] = p.sfw + ((long long)t.expert * p.N + min(t.n0 + r, p.N - 1)) * n_sf;
#pragma unroll
            for (int q = 0; q < C::PK * C::SFB; ++q) {
                const int c = min((q % C::SFB) * 128 + r, C::NB - 1);  // column of the MMA
                const int plane = C::PCOL ? c / C::BT : q / C::SFB, tok = C::PCOL ? c % C::BT : c;
                src[1 + q] = p.sfb + ((long long)plane * p.rows + min(t.row0 + tok, p.rows - 1)) * n_sf;
            }
            const int last = (k1 - 1) >> 2;
            auto load = [&](int q, int grp) {
                return mt_scale_bytes(src[q], 16 * grp, n_sf, p.vec);
            };
            uint4 v[AHEAD][NL];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
#pragma unroll
                for (int q = 0; q < NL; ++q) v[a][q] = load(q, min((k0 >> 2) + a, last));
            for (int base = k0 >> 2; base <= last; base += AHEAD) {
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    if (base + a > last) break;
                    if (!mt_wait(s_empty(g % C::SG), ((uint32_t)(g / C::SG) & 1u) ^ 1u, abort, 16)) break;
                    const uint32_t to = sdst + (g % C::SG) * 4 * C::S_BYTES;
                    ++g;
#pragma unroll
                    for (int q = 0; q < NL; ++q) {
                        const uint32_t w[4] = {v[a][q].x, v[a][q].y, v[a][q].z, v[a][q].w};
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + c * C::S_BYTES + 512 * q), "r"(w[c])
                                         : "memory");
                        v[a][q] = load(q, min(base + a + AHEAD, last));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(scaled((g - 1) % C::SG));
                }
            }
        }
    } else {
        // ---------------- epilogue ----------------
        constexpr int CH = C::BT < 16 ? C::BT : 16;
        const int row = (warp & 3) * 32 + lane;  // weight row of the tile = TMEM lane
        const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        int seg = 0;
        while (walk.next(tile, k0, k1) && !*abort) {
            const MxTile t = mt_tile(p, tile, C::BT);
            const int b = seg % C::ACCS;
            if (!mt_wait(acc_full(b), (uint32_t)(seg / C::ACCS) & 1u, abort, 32)) break;
            ++seg;
            tc_fence_after();
            const bool whole = k0 == 0 && k1 == p.KB;
            const int n = t.n0 + row;
            // a block's first stretch may begin inside a tile, its last may end inside one
            float* part = p.partial + (long long)(2 * blockIdx.x + (k0 == 0)) * (C::BT * MT_ROWS) + row;
            auto store_y = [&](int j, float f) {
                const long long out = p.dst ? (long long)ld_dep(p.dst + t.row0 + j) : t.row0 + j;
                p.y[out * p.N + n] = H::from_f32(f);
            };
#pragma unroll 1
            for (int c0 = 0; c0 < t.rows; c0 += CH) {
                float f[CH];
#pragma unroll
                for (int q = 0; q < (C::PCOL ? C::P : 1); ++q) {
                    uint32_t u[CH];
                    mt_tmem_ld<CH>(t_lane + b * C::NB + q * C::BT + c0, u);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < CH; ++j) f[j] = q ? f[j] + __uint_as_float(u[j]) : __uint_as_float(u[j]);
                }
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    if (c0 + j >= t.rows) continue;
                    if (!whole) part[(c0 + j) * MT_ROWS] = f[j];
                    else if (n < p.N) store_y(c0 + j, f[j]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(b));
            if (whole) continue;
            int first, final_;
            if (!mt_last_of(p, walk, tile, first, final_)) continue;
            for (int c0 = 0; c0 < t.rows; c0 += 8) {
                float f[8];
                const int nj = min(8, t.rows - c0);
                mt_join8(p, first, final_, C::BT, c0, nj, row, f);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < nj && n < p.N) store_y(c0 + j, f[j]);
            }
        }
    }
    if (*abort) __nanosleep(1000000);  // after a wait gave up: let copies in flight land
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
    }
}

// Activations to P e4m3 planes [P][R][K] with scales [P][R][K/32], rows taken
// through `src`; four lanes hold a block.  P = 1 copies mxfp8 rows.  Also
// clears the tile counters of the product that follows and, in a grouped call,
// the y rows whose id has no expert.
template <int T, int P>
__global__ void __launch_bounds__(256) mx_planes_kernel(const void* x, const uint8_t* xs, uint8_t* planes,
                                                        uint8_t* scales, const uint32_t* src, int x_rows, int R, int K,
                                                        uint32_t* counters, int n_counters, const int32_t* ids, int E,
                                                        uint16_t* y, int N) {
    pdl_launch_dependents();
    const long long tid = (long long)blockIdx.x * blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x;
    for (long long i = tid; i < n_counters; i += step) counters[i] = 0;
    if (ids)
        for (long long r = tid >> 5; r < R; r += step >> 5)
            if ((uint32_t)ld_dep(ids + r) >= (uint32_t)E)
                for (int n = threadIdx.x & 31; n < N; n += 32) y[r * N + n] = 0;
    if (!planes) return;
    const int g = K / 8;
    const long long n8 = (long long)R * g;
    for (long long base = tid & ~31LL; base < n8; base += step) {
        const long long i = base + (threadIdx.x & 31);
        const bool in = i < n8;
        const int r = in ? (int)(i / g) : 0, c = (int)(i - (long long)r * g);
        long long from = r;
        if (src && in) from = ld_dep(src + r);
        from = from < x_rows ? from : x_rows - 1;
        if constexpr (P == 1) {
            if (!in) continue;
            const uint2 v = ld_dep(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(x) + from * K) + c);
            reinterpret_cast<uint2*>(planes)[i] = v;
            if ((c & 3) == 0) scales[i >> 2] = ld_dep(xs + from * (K / 32) + (c >> 2));
        } else {
            float v[8] = {};
            if (in) load8<T>(static_cast<const uint16_t*>(x) + from * K + c * 8, v);
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t a = abs_bits(v[j]);
                if (a < 0x7F800000u) m = max(m, a);
                else v[j] = __uint_as_float(0x7FC00000u);  // an infinity has no code: NaN
            }
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            float inv;
            // 128 <= largest < 256 on the grid: rounding cannot reach 448
            uint32_t byte = mx_scale_byte<7>(m, inv);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inv;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = cvt2_e4m3(v[2 * j], v[2 * j + 1]);
                if (in) {
                    const long long o = (long long)q * n8 + i;
                    reinterpret_cast<uint2*>(planes)[o] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
                    if ((c & 3) == 0) scales[o >> 2] = (uint8_t)byte;
                }
                if (q + 1 < P) {
                    const uint32_t next = byte > 4 ? byte - 4 : 0;  // the remainder, up to 16 times larger
                    const float up = __uint_as_float((127u + byte - next) << 23);
                    byte = next;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t f = e4m3x2_f16x2(h[j]);
                        v[2 * j] = (v[2 * j] - Half<true>::lo_f32(f)) * up;
                        v[2 * j + 1] = (v[2 * j + 1] - Half<true>::hi_f32(f)) * up;
                    }
                }
            }
        }
    }
}

}  // namespace qmm

namespace qmm_host {

namespace {

// Workspace of a tensor-core product behind the row tables.
struct TcLayout {
    size_t planes, scales, counters, partial, bytes;
    bool prep;
};

int planes_of(bool mx, bool f16) { return mx ? 1 : f16 ? 3 : 2; }

long long tiles_max(long long rows, long long E, long long N, int bt, bool grouped) {
    const long long items = grouped ? rows / bt + (E < rows ? E : rows) + 1 : (rows + bt - 1) / bt;
    return items * ((N + 127) / 128);
}

// Whether the k-blocks of the tiles are divided over the blocks: with fewer
// whole tiles than about eight for each block the last round of tiles would
// leave many blocks without one.
bool tc_split(long long tiles, int bt) { return bt <= 64 ? tiles < 8 * kMxMaxBlocks : tiles < kMxMaxBlocks; }

TcLayout tc_layout(long long rows, long long E, long long N, long long K, bool mx, bool f16, bool grouped, int bt) {
    TcLayout l{};
    const long long tiles = tiles_max(rows, E, N, bt, grouped);
    const bool split = tc_split(tiles, bt);
    l.prep = !mx || grouped;  // mxfp8 rows of a dense call are read where they are
    const int P = planes_of(mx, f16);
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t o = at;
        at += mx_al256(n);
        return o;
    };
    l.planes = take(l.prep ? (size_t)P * rows * K : 0);
    l.scales = take(l.prep ? (size_t)P * rows * (K / 32) : 0);
    l.counters = take(split ? (size_t)tiles * 16 : 0);
    l.partial = take(split ? (size_t)2 * kMxMaxBlocks * bt * 128 * 4 : 0);
    l.bytes = at;
    return l;
}

template <class C>
int launch_tc(const MxMatmul& a, const CUtensorMap& mw, const CUtensorMap& mb, const qmm::MxTcParams& p, int blocks,
              bool pdl) {
    auto kern = qmm::mx_tc_kernel<C>;
    int rc = ensure_smem_limit((const void*)kern, C::SMEM, "mx_tc smem attribute");
    if (rc) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = a.st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = pdl && pdl_enabled() ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, kern, mw, mb, p), "mx_tc launch");
}

template <bool F16, int P>
int launch_tc_bt(const MxMatmul& a, const CUtensorMap& mw, const CUtensorMap& mb, const qmm::MxTcParams& p, int blocks,
                 bool pdl, int bt) {
    using namespace qmm;
    if constexpr (P == 2)
        if (bt == 8) return launch_tc<MxTc<F16, P, true, 8, 11>>(a, mw, mb, p, blocks, pdl);
    if (bt == 16) return launch_tc<MxTc<F16, P, true, 16, P == 3 ? 9 : P == 2 ? 10 : 11>>(a, mw, mb, p, blocks, pdl);
    if (bt == 64) return launch_tc<MxTc<F16, P, true, 64, P == 1 ? 8 : P == 2 ? 6 : 5>>(a, mw, mb, p, blocks, pdl);
    if (bt == 128) return launch_tc<MxTc<F16, P, false, 128, P == 1 ? 6 : P == 2 ? 4 : 3>>(a, mw, mb, p, blocks, pdl);
    if constexpr (P < 3) return launch_tc<MxTc<F16, P, false, 256, P == 1 ? 4 : 2>>(a, mw, mb, p, blocks, pdl);
    set_error("mx_tc: no tile of %d rows", bt);
    return QMM_EUNSUPPORTED;
}

}  // namespace

// Rows of a tile: the narrowest that takes all rows of an expert (on average)
// in one, since every tile reads its weights again.
int mx_tc_item_rows(long long rows, long long E, bool mx, bool f16) {
    const long long mean = (rows + E - 1) / E;
    if (mean <= 8 && planes_of(mx, f16) == 2) return 8;
    if (mean <= 16) return 16;
    if (mean <= 64) return 64;
    return mean <= 128 || planes_of(mx, f16) == 3 ? 128 : 256;
}

// TMA spreads the codes in runs of 128 from 32-byte aligned rows; scale words
// are four bytes.
bool mx_tc_takes(const void* x, const uint8_t* xs, const uint32_t* w, const uint8_t* ws, long long rows, long long E,
                 long long N, long long K) {
    return K % 128 == 0 && ((uintptr_t)w & 31u) == 0 && ((uintptr_t)ws & 3u) == 0 && ((uintptr_t)xs & 3u) == 0 &&
           E * N <= (1LL << 31) - 256 && 3 * rows <= (1LL << 31) - 256;
}

size_t mx_tc_workspace(long long rows, long long E, long long N, long long K, bool mx, bool f16, bool grouped) {
    return tc_layout(rows, E, N, K, mx, f16, grouped, mx_tc_item_rows(rows, E, mx, f16)).bytes;
}

int launch_mx_tc(const MxMatmul& a, const int4* items, const int32_t* n_items, const int32_t* ids, int bt, void* ws) {
    const bool mx = a.xs != nullptr, grouped = items != nullptr;
    const int P = planes_of(mx, a.f16);
    const TcLayout l = tc_layout(a.rows, a.E, a.N, a.K, mx, a.f16, grouped, bt);
    char* const base = static_cast<char*>(ws);
    const long long tiles = tiles_max(a.rows, a.E, a.N, bt, grouped);
    qmm::MxTcParams p{};
    p.split = tc_split(tiles, bt);
    uint8_t* planes = reinterpret_cast<uint8_t*>(base + l.planes);
    uint8_t* scales = reinterpret_cast<uint8_t*>(base + l.scales);
    uint32_t* counters = reinterpret_cast<uint32_t*>(base + l.counters);
    p.sfw = a.ws;
    p.sfb = l.prep ? scales : a.xs;
    p.y = static_cast<uint16_t*>(a.y);
    p.items = items;
    p.n_items = n_items;
    p.dst = a.dst;
    p.partial = reinterpret_cast<float*>(base + l.partial);
    p.counters = counters;
    p.rows = (int)a.rows;
    p.K = (int)a.K;
    p.N = (int)a.N;
    p.KB = (int)(a.K / 128);
    p.n_tiles = (int)((a.N + 127) / 128);
    p.vec = mx_scale_vec(a.K, p.sfw, p.sfb);
    const long long units = tiles * p.KB;
    const int sms = mx_sm_count();
    int blocks = (int)(tiles < sms ? tiles : sms);
    if (p.split) {  // at least four k-blocks each: a join reads every sharer's part
        const long long most = (units + 3) / 4;
        blocks = (int)(most < sms ? most : sms);
    }

    const bool prep = l.prep || p.split;
    if (prep) {
        const long long n8 = l.prep ? a.rows * (a.K / 8) : 1;
        const long long want = (n8 + 255) / 256;
        const unsigned g = (unsigned)(want < 148 * 8 ? want : 148 * 8);
        const int nc = p.split ? (int)tiles * 4 : 0;
        uint8_t* out = l.prep ? planes : nullptr;
#define QMM_PLANES(T, PP)                                                                                          \
    qmm::mx_planes_kernel<T, PP><<<g, 256, 0, a.st>>>(a.x, a.xs, out, scales, a.src, (int)a.x_rows, (int)a.rows,    \
                                                      (int)a.K, counters, nc, ids, (int)a.E, p.y, (int)a.N)
        if (mx) QMM_PLANES(qmm::MX_BF16, 1);
        else if (a.f16) QMM_PLANES(qmm::MX_F16, 3);
        else QMM_PLANES(qmm::MX_BF16, 2);
#undef QMM_PLANES
        const int rc = cuda_status(cudaGetLastError(), "mx_planes launch");
        if (rc) return rc;
    }
    CUtensorMap mw, mb;
    int rc = tensor_map_2d(&mw, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, a.w, (uint64_t)a.K, (uint64_t)(a.E * a.N),
                           (uint64_t)a.K / 2, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = tensor_map_2d(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, l.prep ? planes : a.x, (uint64_t)a.K,
                       (uint64_t)(P * a.rows), (uint64_t)a.K, 128, (uint32_t)bt, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    if (mx) return a.f16 ? launch_tc_bt<true, 1>(a, mw, mb, p, blocks, prep, bt)
                         : launch_tc_bt<false, 1>(a, mw, mb, p, blocks, prep, bt);
    return a.f16 ? launch_tc_bt<true, 3>(a, mw, mb, p, blocks, prep, bt)
                 : launch_tc_bt<false, 2>(a, mw, mb, p, blocks, prep, bt);
}

int mx_tc_device_error(int reset) { return mx_error_flag(reset); }

}  // namespace qmm_host
