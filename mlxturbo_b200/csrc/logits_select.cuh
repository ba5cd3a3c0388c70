// logits_select.cuh -- selection in a row of logits: a cluster's candidates
// for the largest tokens, and the border key of any count or mass.
#pragma once

#include "logits.cuh"
#include "search.cuh"

namespace qmm {

// Bins of a row's mass.
constexpr int kBins = 512;

// A cluster's candidates are in its CTA 0.
struct DrawShared {  // of a draw without filters
    double slots[2][kMaxRowWarps];
    WarpStat stats[kMaxRowWarps];
    FindShared find;
    double table[32];  // of Weight64
    int verdict;
};

struct SelectShared : DrawShared {
    union {
        struct {
            union {
                float maxima[kRowThreads * kMaxCluster];  // of groups of lanes of the cluster
                double w[kCand];                          // the sorted candidates' weights
                uint32_t piv_count[2][kMaxRowWarps][8];
            };
            union {
                unsigned long long cand[kCand];  // CTA 0's copy is used
                double piv_mass[2][kMaxRowWarps][8];
            };
        };
        uint32_t bins[kRowWarps][2][kBins];  // of each warp: masses in two limbs
    };
    unsigned long long bin_sum[kBins];
    uint32_t found[kMaxRowWarps];
    uint32_t hist[256];
    uint32_t n_cand, sel_bin, sel_above;
    unsigned long long bin_above, best;
    double scan[kRowWarps];
};

constexpr size_t kSelectSmem = sizeof(SelectShared) + kRing * kRowThreads * sizeof(uint4);
constexpr size_t kDrawSmem = sizeof(DrawShared) + kRing * kRowThreads * sizeof(uint4);

// The largest 16-bit prefix b such that at least k of the n maxima have
// key32 >> 16 >= b; 0 if there are fewer than k.  One CTA, all threads.
QMM_DEVINL uint32_t kth_prefix(SelectShared& sh, int n, int k) {
    uint32_t prefix = 0;
    int left = k;
    for (int level = 0; level < 2; ++level) {
        for (int i = threadIdx.x; i < 256; i += kRowThreads) sh.hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kRowThreads) {
            const uint32_t p = key32(sh.maxima[i]) >> 16;
            if (level == 0) atomicAdd(&sh.hist[p >> 8], 1u);
            else if ((p >> 8) == prefix) atomicAdd(&sh.hist[p & 255u], 1u);
        }
        __syncthreads();
        // warp 0: the bin, from the top, at which the count reaches `left`
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x;
            uint32_t h[8], run = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[i] = sh.hist[255 - (lane * 8 + i)];
                run += h[i];
            }
            uint32_t incl = run;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(~0u, incl, o);
                if (lane >= o) incl += y;
            }
            const unsigned hits = __ballot_sync(~0u, incl >= (uint32_t)left);
            if (hits == 0) {
                if (lane == 0) sh.sel_bin = 0xFFFFFFFFu;  // fewer than `left`
            } else if (lane == __ffs(hits) - 1) {
                uint32_t before = incl - run;
                bool done = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (!done && before + h[i] >= (uint32_t)left) {
                        sh.sel_bin = 255 - (lane * 8 + i);
                        sh.sel_above = before;
                        done = true;
                    }
                    if (!done) before += h[i];
                }
            }
        }
        __syncthreads();
        const uint32_t b = sh.sel_bin, above = sh.sel_above;
        __syncthreads();
        if (b == 0xFFFFFFFFu) return 0;
        prefix = (prefix << 8) | b;
        left -= (int)above;
    }
    return prefix;
}

// How many lanes share one published maximum: the k-th largest of the maxima
// bounds the k-th largest logit from below, and with at least twice as many
// maxima as k about 1.4 k logits reach it.  Few maxima are searched by every
// warp on its own.
QMM_DEVINL int lanes_to_group(int warps, int k) {
    int lanes = 32;
    while (lanes > 1 && warps * (32 / lanes) < 2 * k) lanes >>= 1;
    return lanes;
}

// The maxima of a warp's groups to every CTA of the cluster.
QMM_DEVINL void publish_maxima(cg::cluster_group& cl, SelectShared& sh, int g, int lanes, float top) {
    const int lane = threadIdx.x & 31;
    for (int o = 1; o < lanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    if (lane % lanes == 0) {
        float* to = sh.maxima + g * (32 / lanes) + lane / lanes;
        for (int i = 0; i < (int)cl.num_blocks(); ++i) *cl.map_shared_rank(to, i) = top;
    }
}

// key32 of a bound that at least k of the n maxima reach (0: fewer than k are
// there).  Up to 256 maxima by each warp on its own, else by the CTA together.
template <int PER>
QMM_DEVINL uint32_t kth_of_warp(const float* maxima, int n, int k) {
    const int lane = threadIdx.x & 31;
    uint32_t key[PER], most = 0, least = 0xFFFFu;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        key[i] = i * 32 + lane < n ? key32(maxima[i * 32 + lane]) >> 16 : 0;
        most = max(most, key[i]);
        least = min(least, key[i]);
    }
    // bit by bit, below the bits that all keys share: the largest prefix that k keys reach
    const uint32_t all = __reduce_max_sync(~0u, most), differ = all ^ __reduce_min_sync(~0u, least);
    uint32_t bit = differ ? 0x80000000u >> __clz(differ) : 0, b = bit ? all & ~(2 * bit - 1) : all;
    for (; bit; bit >>= 1) {
        int reach = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) reach += __popc(__ballot_sync(~0u, key[i] >= (b | bit)));
        if (reach >= k) b |= bit;
    }
    return b << 16;
}

QMM_DEVINL uint32_t kth_bound(SelectShared& sh, int n, int k) {
    if (n < k) return 0;
    if (n <= 128) return kth_of_warp<4>(sh.maxima, n, k);
    if (n <= 256) return kth_of_warp<8>(sh.maxima, n, k);
    return kth_prefix(sh, n, k) << 16;
}

// The tokens of K vectors to a lane that `take` wants to CTA 0's list, in any
// order.  By a whole warp; v < 0: none.  The list's count may pass kCand; no
// more than that are written.  Returns the warp's number.
template <int DT, int K, typename F>
QMM_DEVINL uint32_t append_if(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const int (&v)[K],
                              const uint4 (&u)[K], F&& take) {
    constexpr int N = Elem<DT>::kVec;
    const int lane = threadIdx.x & 31;
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        float x[N];
        decode<DT>(u[i], x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int id = row.first(v[i]) + j;
            if (v[i] >= 0 && id >= 0 && id < row.V && take(id, x[j])) hit |= 1u << (i * N + j);
        }
    }
    if (!__any_sync(~0u, hit != 0)) return 0;
    const uint32_t mine = __popc(hit);
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += y;
    }
    const uint32_t total = __shfl_sync(~0u, incl, 31);
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(cl.map_shared_rank(&sh.n_cand, 0), total);
    at = __shfl_sync(~0u, at, 0) + incl - mine;
    unsigned long long* list = cl.map_shared_rank(sh.cand, 0);
#pragma unroll
    for (int i = 0; i < K; ++i) {
        float x[N];
        decode<DT>(u[i], x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!(hit >> (i * N + j) & 1)) continue;
            if (at < kCand) list[at] = row_key(x[j], row.first(v[i]) + j);
            ++at;
        }
    }
    return total;
}

template <int DT, typename F>
QMM_DEVINL uint32_t append_if(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, int v, const uint4& u,
                              F&& take) {
    const int vs[1] = {v};
    const uint4 us[1] = {u};
    return append_if<DT, 1>(cl, sh, row, vs, us, take);
}

// Those with key32 in [lo, hi) and key >= floor.
template <int DT, int K>
QMM_DEVINL uint32_t append(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const int (&v)[K],
                           const uint4 (&u)[K], uint32_t lo, uint32_t hi, unsigned long long floor) {
    return append_if<DT, K>(cl, sh, row, v, u, [&](int id, float x) {
        const uint32_t k = key32(x);
        return k >= lo && k < hi && row_key(x, id) >= floor;
    });
}

// The same over the whole slice.  A lane keeps up to four tokens until the end,
// so that a warp reserves its places once (a round trip to CTA 0 is 1 us, and
// hits come in most turns of the loop); where a lane meets more, vector by vector.
template <int DT, typename F>
QMM_DEVINL uint32_t append_slice(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s,
                                 F&& take) {
    constexpr int N = Elem<DT>::kVec, kKeep = 4;
    const int first = s.head >= 0 ? s.head : s.begin, last = s.tail >= 0 ? s.tail + 1 : s.end;
    auto each = [&](auto&& f) {
        for (int v0 = first; v0 < last; v0 += 128) {
            uint4 u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = v0 + 32 * i + s.lane;
                u[i] = v < last ? row.load(v) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) f(v0 + 32 * i + s.lane, u[i]);
        }
    };
    unsigned long long key[kKeep] = {};
    uint32_t mine = 0;
    each([&](int v, const uint4& u) {
        if (v >= last) return;
        float x[N];
        decode<DT>(u, x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int id = row.first(v) + j;
            if (id < 0 || id >= row.V || !take(id, x[j])) continue;
#pragma unroll
            for (int i = 0; i < kKeep; ++i)
                if (mine == (uint32_t)i) key[i] = row_key(x[j], id);
            ++mine;
        }
    });
    uint32_t found = 0;
    if (__any_sync(~0u, mine > kKeep)) {
        each([&](int v, const uint4& u) { found += append_if<DT>(cl, sh, row, v < last ? v : -1, u, take); });
        return found;
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, incl, o);
        if (s.lane >= o) incl += y;
    }
    found = __shfl_sync(~0u, incl, 31);
    if (!found) return 0;
    uint32_t at = 0;
    if (s.lane == 0) at = atomicAdd(cl.map_shared_rank(&sh.n_cand, 0), found);
    at = __shfl_sync(~0u, at, 0) + incl - mine;
    unsigned long long* list = cl.map_shared_rank(sh.cand, 0);
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
        if ((uint32_t)i < mine && at + i < kCand) list[at + i] = key[i];
    return found;
}

// Those with key32 in [lo, hi) and key >= floor.
template <int DT>
QMM_DEVINL uint32_t append_slice(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s,
                                 uint32_t lo, uint32_t hi, unsigned long long floor) {
    return append_slice<DT>(cl, sh, row, s, [&](int id, float x) {
        const uint32_t k = key32(x);
        return k >= lo && k < hi && row_key(x, id) >= floor;
    });
}

// Candidates: every token with key32 >= bound.  A lane reads its two vectors
// of the largest maxima again, as far as they reach the bound; one where a third
// may reach it has all of its vectors (begin + owner, begin + owner + 32, .., and
// lane 0 the row's ends) read by the warp.  What is read is read at once: under a
// busy memory every wait here is 2 us.
template <int DT>
QMM_DEVINL uint32_t push_candidates(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s,
                                    const LaneTop& top, uint32_t bound) {
    const bool more = key32(top.others) >= bound;
    unsigned owners = __ballot_sync(~0u, more);
    if (__popc(owners) > 6) return append_slice<DT>(cl, sh, row, s, bound, 0xFFFFFFFFu, 0);
    const int v[2] = {!more && key32(top.first) >= bound ? top.at : -1,
                      !more && key32(top.second) >= bound ? top.at2 : -1};
    uint4 u[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) u[i] = v[i] >= 0 ? row.load(v[i]) : make_uint4(0, 0, 0, 0);
    uint32_t found = append<DT, 2>(cl, sh, row, v, u, bound, 0xFFFFFFFFu, 0);
    while (owners) {
        const int owner = __ffs(owners) - 1;
        owners &= owners - 1;
        for (int v0 = s.begin + owner; v0 < s.end; v0 += 64 * 32) {
            const int w[2] = {v0 + 32 * s.lane < s.end ? v0 + 32 * s.lane : -1,
                              v0 + 32 * (s.lane + 32) < s.end ? v0 + 32 * (s.lane + 32) : -1};
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (w[i] >= 0) u[i] = row.load_whole(w[i]);
            found += append<DT, 2>(cl, sh, row, w, u, bound, 0xFFFFFFFFu, 0);
        }
        if (owner == 0) {
            const int w[1] = {s.lane == 0 ? s.head : s.lane == 1 ? s.tail : -1};
            const uint4 end[1] = {w[0] >= 0 ? row.load(w[0]) : make_uint4(0, 0, 0, 0)};
            found += append<DT, 1>(cl, sh, row, w, end, bound, 0xFFFFFFFFu, 0);
        }
    }
    return found;
}

// Descending sort of the first n candidates (distinct keys) in place, above 256
// bitonic, padded with 0, which no token's key is.  One CTA, in step before it.
QMM_DEVINL void sort_candidates(unsigned long long* k, int n) {
    if (n <= kRowThreads) {  // a thread to a key: its place is the number of larger ones
        const unsigned long long mine = (int)threadIdx.x < n ? k[threadIdx.x] : 0;
        int place = 0;
        for (int i = 0; i < n; ++i) place += k[i] > mine;
        __syncthreads();
        if ((int)threadIdx.x < n) k[place] = mine;
        __syncthreads();
        return;
    }
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kRowThreads) k[i] = 0;
    __syncthreads();
    for (int span = 2; span <= size; span <<= 1) {
        for (int step = span / 2; step >= 1; step >>= 1) {
            for (int t = threadIdx.x; t < size / 2; t += kRowThreads) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const unsigned long long a = k[i], b = k[j];
                if ((a < b) == ((i & span) == 0)) {
                    k[i] = b;
                    k[j] = a;
                }
            }
            __syncthreads();
        }
    }
}

// The CTA's sum, the same in every thread.
QMM_DEVINL double cta_sum(SelectShared& sh, double x) {
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.scan[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0.0;
    for (int i = 0; i < kRowWarps; ++i) x += sh.scan[i];
    return x;
}

// Running sums over the sorted candidates' weights, in place, by the whole CTA.
QMM_DEVINL void scan_weights(SelectShared& sh, int n) {
    const int per = (n + kRowThreads - 1) / kRowThreads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = threadIdx.x * per, e = b + per < n ? b + per : n;
    double run = 0.0;
    for (int i = b; i < e; ++i) run += sh.w[i];
    double incl = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) sh.scan[warp] = incl;
    __syncthreads();
    double base = incl - run;
    for (int i = 0; i < warp; ++i) base += sh.scan[i];
    for (int i = b; i < e; ++i) {
        base += sh.w[i];
        sh.w[i] = base;
    }
    __syncthreads();
}

// ---- borders by search -------------------------------------------------------------
//
// The border of a count or a mass: the first token of the order at which the
// tokens from the top on, of those with keys >= floor, reach it.  Rounds of one
// pass each: eight pivots cut the range that holds the border, and only tokens
// within the range are counted and weighed (in 64 bits); from the second round
// on that is a small part of them.  Once few enough are left they go to CTA 0,
// which sorts them and runs through them.
//
// kInRange: sorting 512 costs about as much as one more round.
constexpr uint32_t kInRange = 512;

// A pivot between two logits' values, in the order of keys.
QMM_DEVINL uint32_t between(uint32_t lo, uint32_t hi, int j, bool by_value) {
    const uint32_t step = (hi - lo) / 8, even = lo + (step > 0 ? step * j : j);
    if (!by_value) return even;
    const float a = key32_value(lo), b = key32_value(hi);
    const float v = a + (b - a) * (0.125f * j);
    const uint32_t k = key32(v);  // NaN (infinite ends): kKeyNegInf, which the caller clamps
    return k > lo && k < hi ? k : even;
}

// MASS: `want` is a part of the mass of all tokens >= floor, else a count.
// Returns the border key; floor if the tokens do not reach it.  All threads of
// the cluster; every thread returns the same.
template <int DT, bool MASS>
QMM_DEVINL unsigned long long border_key(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s,
                                         int g, int warps, Ring ring, const Weight64& weight,
                                         unsigned long long floor, double want) {
    constexpr int N = Elem<DT>::kVec;
    const int rank = (int)cl.block_rank();
    uint32_t lo = (uint32_t)(floor >> 32), hi = key32(weight.mx) + 1, inside = 0xFFFFFFFFu;
    double above = 0.0, target = want;  // measure of the keys from hi on
    cl.sync();                          // the shared arrays' earlier readers
    for (int round = 0; round == 0 || (hi - lo > 1 && inside > kInRange); ++round) {
        // pivot 0 is lo; the first round looks where weights are, later ones cut values, or keys, evenly
        uint32_t p[8];
        p[0] = lo;
#pragma unroll
        for (int j = 1; j < 8; ++j) {
            if (round == 0 && MASS) {
                // 24, 16, 11, 8, 5.5, 3.5, 1.5 temperatures below the maximum
                const float depth = j == 1 ? 24.f : j == 2 ? 16.f : j == 3 ? 11.f : j == 4 ? 8.f : j == 5 ? 5.5f
                                    : j == 6 ? 3.5f : 1.5f;
                p[j] = key32(weight.mx - depth / (float)weight.inv_t);
            } else {
                p[j] = between(lo, hi, j, round < 8 && (round & 1) == (MASS ? 1 : 0));
            }
            p[j] = max(p[j], p[j - 1]);
            p[j] = min(p[j], hi);
        }
        uint32_t n[8];
        double m[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            n[j] = 0;
            m[j] = 0.0;
        }
        for_vectors_slow<DT>(row, s, ring, [&](int v, const uint4& u) {
            float x[N];
            uint32_t k[N];
            bool any = false;
            decode<DT>(u, x);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int id = row.first(v) + e;
                k[e] = key32(x[e]);
                const bool in = k[e] >= lo && k[e] < hi && id >= 0 && id < row.V && row_key(x[e], id) >= floor;
                if (!in) k[e] = 0;  // below every pivot
                any |= in;
            }
            if (!any) return;
            double w[N];
            if (MASS) {
#pragma unroll
                for (int e = 0; e < N; ++e) w[e] = weight(x[e]);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (k[e] >= p[j]) {
                        ++n[j];
                        if (MASS) m[j] += w[e];
                    }
                }
            }
        });
        const int buf = round & 1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            n[j] = warp_sum(n[j]);
            if (MASS) m[j] = warp_sum(m[j]);
        }
        if (s.lane < (int)cl.num_blocks()) {
            uint32_t* pn = cl.map_shared_rank(sh.piv_count[buf][g], s.lane);
            double* pm = cl.map_shared_rank(sh.piv_mass[buf][g], s.lane);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                pn[j] = n[j];
                if (MASS) pm[j] = m[j];
            }
        }
        cl.sync();
        // lanes j, j + 8, .. of every warp: pivot j's totals, in a fixed order
        uint32_t tn = 0;
        double tm = 0.0;
        for (int i = s.lane >> 3; i < warps; i += 4) {
            tn += sh.piv_count[buf][i][s.lane & 7];
            if (MASS) tm += sh.piv_mass[buf][i][s.lane & 7];
        }
#pragma unroll
        for (int o = 8; o <= 16; o <<= 1) {
            tn += __shfl_xor_sync(~0u, tn, o);
            if (MASS) tm += __shfl_xor_sync(~0u, tm, o);
        }
        const double got = above + (MASS ? tm : (double)tn);
        if (round == 0 && MASS) target = fmax(want * __shfl_sync(~0u, got, 0), 1e-300);
        unsigned reached = __ballot_sync(~0u, got >= target) & 0xFFu;
        if (round == 0 && !(reached & 1u)) return floor;  // not even all of them
        reached |= 1u;  // lo was found to reach it: sums cut otherwise may fall short of that by their last bits
        const int at = 31 - __clz(reached), nxt = at < 7 ? at + 1 : 7;
        const uint32_t n_at = __shfl_sync(~0u, tn, at), n_next = __shfl_sync(~0u, tn, nxt);
        const double got_next = __shfl_sync(~0u, got, nxt);
        uint32_t p_at = p[0], p_next = hi;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j == at) p_at = p[j];
            if (j == at + 1) p_next = p[j];
        }
        lo = p_at;
        inside = n_at;
        if (at < 7) {
            hi = p_next;
            inside -= n_next;
            above = got_next;
        }
    }
    if (inside > kInRange) {
        // one logit's value, more often than the list is long: the first of them by id.  Equal weights: a count.
        const double w = weight(key32_value(lo));
        double need = target - above;
        if (MASS) {  // a quotient rounds, and is no number where w is 0
            const double guess = fmin(fmax(ceil(need / w), 1.0), (double)inside);
            need = (double)lowest_kept(1, inside, (uint32_t)guess, [&](uint32_t n) { return above + n * w >= target; });
        }
        unsigned long long a = (unsigned long long)lo << 32, b = (unsigned long long)(lo + 1) << 32;
        if (floor > a) a = floor;
        for (int round = 0; b - a > 1; ++round) {  // the largest key with `need` tokens from it on
            const unsigned long long step = (b - a) / 8 > 0 ? (b - a) / 8 : 1;
            uint32_t n[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) n[j] = 0;
            for_vectors_slow<DT>(row, s, ring, [&](int v, const uint4& u) {
                float x[N];
                decode<DT>(u, x);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int id = row.first(v) + e;
                    if (key32(x[e]) != lo || id < 0 || id >= row.V) continue;
                    const unsigned long long k = row_key(x[e], id);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (k >= a + j * step) ++n[j];
                }
            });
            const int buf = round & 1;
            if (round == 0) cl.sync();
#pragma unroll
            for (int j = 0; j < 8; ++j) n[j] = warp_sum(n[j]);
            if (s.lane < (int)cl.num_blocks()) {
                uint32_t* pn = cl.map_shared_rank(sh.piv_count[buf][g], s.lane);
#pragma unroll
                for (int j = 0; j < 8; ++j) pn[j] = n[j];
            }
            cl.sync();
            uint32_t tn = 0;
            for (int i = s.lane >> 3; i < warps; i += 4) tn += sh.piv_count[buf][i][s.lane & 7];
#pragma unroll
            for (int o = 8; o <= 16; o <<= 1) tn += __shfl_xor_sync(~0u, tn, o);
            const unsigned reached =
                __ballot_sync(~0u, a + (s.lane & 7) * step < b && (double)tn >= need) & 0xFFu;
            if (!(reached & 1u)) return a;
            const int at = 31 - __clz(reached);
            const unsigned long long from = a;
            a = from + at * step;
            if (at < 7 && from + (at + 1) * step < b) b = from + (at + 1) * step;
        }
        return a;
    }
    // the tokens left, in order
    cl.sync();
    if (rank == 0 && threadIdx.x == 0) sh.n_cand = 0;
    cl.sync();
    append_slice<DT>(cl, sh, row, s, lo, hi, floor);
    cl.sync();
    if (rank == 0) {
        const int n = (int)sh.n_cand;
        sort_candidates(sh.cand, n);
        if (MASS) {
            for (int i = threadIdx.x; i < n; i += kRowThreads) sh.w[i] = weight(key32_value((uint32_t)(sh.cand[i] >> 32)));
            __syncthreads();
            scan_weights(sh, n);
        }
        int first = MASS ? n - 1 : (int)(target - above) - 1;  // the token at which the target is reached
        if (MASS) {
            int b = 0, e = n - 1;
            while (b < e) {
                const int mid = (b + e) / 2;
                if (above + sh.w[mid] >= target) e = mid;
                else b = mid + 1;
            }
            first = b;
        }
        if (threadIdx.x < cl.num_blocks()) *cl.map_shared_rank(&sh.best, threadIdx.x) = sh.cand[first];
    }
    cl.sync();
    return sh.best;
}

// ---- the border of a mass by bins ------------------------------------------------------
//
// Most rows with top-p that are not done from the list are open ones: thousands
// of tokens are kept.  One pass weighs every token in 64 bits.  Those below
// `bound` (all but some hundreds) go into bins of equal depth, as whole numbers
// of 2^-40 of the weight there; each warp has bins of its own, in two limbs of
// 20 bits, so that 32-bit adds do for fewer than 4096 tokens to a warp, and a
// sum of whole numbers is the same in any order.  A token is off by half such a
// unit, so a bin's sums, a mass above a bin and a part of the whole by half a
// unit for each token: a border or a draw nearer than that is made in 64 bits
// (V units are 2^-21 of the weight at the edge for V 248320, kept tokens weigh
// a hundredth of it and more: by estimate one row in 10^4 or fewer).  The bins
// reach down to where what is left, V tokens at most, is half of what top-p
// leaves out.  The tokens of the bin that holds the border, less than a
// hundredth of them, go to CTA 0's list.  What lies above it of each warp is
// kept for the draw, so no token is weighed twice.  (128 rows of 248320 at top-p 0.95, half of them open: 411 us
// with border_key's rounds.)

constexpr double kBinMagic = 4503599627370496.0;  // 2^52: a sum with it is a whole number
constexpr int kBinTokens = 4095;                  // of a warp

// The k-th token of the order, by counts in bins between the maximum and half
// again as deep as `low`, the lowest of all lanes' maxima.  Returns false where
// the bins do not reach it or the list does not hold its bin.  (300 rows of
// 248320, k 5000, top-p 0.95: 1774 us with border_key's rounds.)
template <int DT>
QMM_DEVINL bool kth_by_bins(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s, float mx,
                            float low, int k, unsigned long long& border) {
    constexpr int N = Elem<DT>::kVec;
    const int rank = (int)cl.block_rank(), warp = threadIdx.x >> 5, t = threadIdx.x, C = (int)cl.num_blocks();
    const float range = 1.5f * (mx - low);
    if (!(range > 0.0f && range < CUDART_INF_F)) return false;
    const float scale = (float)kBins / range;
    auto bin_of = [&](float x) {  // kBins: below them all, masked or no number
        const float d = (mx - x) * scale;
        return d < (float)kBins ? (int)d : kBins;
    };
    cl.sync();  // the shared arrays' earlier readers
    uint32_t* const count = sh.bins[warp][0];
    for (int i = s.lane; i < kBins; i += 32) count[i] = 0;
    if (t == 0) {
        sh.n_cand = 0;
        sh.sel_bin = kBins;
    }
    __syncwarp();
    for_vectors<DT>(row, s, [&](int, const uint4& u) {
        float x[N];
        decode<DT>(u, x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int bin = bin_of(x[j]);
            if (bin < kBins) atomicAdd(&count[bin], 1u);
        }
    });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        unsigned long long mine = 0;
        for (int w = 0; w < kRowWarps; ++w) mine += sh.bins[w][0][2 * t + i];
        sh.bin_sum[2 * t + i] = mine;
    }
    cl.sync();
    unsigned long long all[2] = {0, 0};
    for (int i = 0; i < C; ++i) {
        const unsigned long long* from = cl.map_shared_rank(sh.bin_sum, i);
        all[0] += from[2 * t];
        all[1] += from[2 * t + 1];
    }
    unsigned long long incl = all[0] + all[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(~0u, incl, o);
        if (s.lane >= o) incl += y;
    }
    unsigned long long* const parts = reinterpret_cast<unsigned long long*>(sh.scan);
    if (s.lane == 31) parts[warp] = incl;
    __syncthreads();
    for (int i = 0; i < warp; ++i) incl += parts[i];
    const unsigned long long mid = incl - all[1], first = mid - all[0], want = (unsigned long long)k;
    if (first < want && incl >= want) {
        sh.sel_bin = (uint32_t)(2 * t + (mid < want));
        sh.bin_above = mid < want ? mid : first;
    }
    __syncthreads();
    const int bin = (int)sh.sel_bin;
    if (bin == kBins) return false;
    const int place = (int)(want - sh.bin_above) - 1;  // in the bin
    cl.sync();                                         // bins and sums are read; the list takes their place
    append_slice<DT>(cl, sh, row, s, [&](int, float x) { return bin_of(x) == bin; });
    cl.sync();
    if (rank == 0) {
        const int n = (int)sh.n_cand;
        const bool ok = n > place && n <= kCand;
        if (ok) sort_candidates(sh.cand, n);
        if (t < C) {
            if (ok) *cl.map_shared_rank(&sh.best, t) = sh.cand[place];
            *cl.map_shared_rank(&sh.verdict, t) = ok;
        }
    }
    cl.sync();
    border = sh.best;
    return sh.verdict != 0;
}

// Border of the part `p` of the mass of the tokens with keys >= floor, `tokens` of
// them at most.  Tokens from `edge` on are summed beside the bins, which reach
// `deep` temperatures below it.  Returns false where bins do not give it: it lies
// above the edge, in the last bin, in one with more tokens than the list holds
// (equal ones), or nearer to a token's end than their sums are.  Else `border` is
// it, and slots[g] in CTA 0 (only) the mass of warp g's tokens from it on; slots
// is a shared array for all warps.  Sums of them, and parts of their whole, are
// off by `slack` together at most.
template <int DT>
QMM_DEVINL bool border_by_bins(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s, int g,
                               int warps, Ring ring, const Weight64& weight, double p, float edge, double deep,
                               unsigned long long floor, int tokens, double* slots, unsigned long long& border,
                               double& slack) {
    constexpr int N = Elem<DT>::kVec;
    const int rank = (int)cl.block_rank(), warp = threadIdx.x >> 5, t = threadIdx.x, C = (int)cl.num_blocks();
    const double w_edge = weight(edge);
    if (!(w_edge > 1e-250) || !(deep > 0.0) || !(deep < 1e3)) return false;
    const float scale = (float)((kBins - 1) * weight.inv_t / deep);
    const double unit = exp2(ceil(log2(w_edge)) - 40.0), per_unit = 1.0 / unit;
    slack = (double)tokens * unit;  // half a unit a token on either side of a comparison
    const float floor_value = key32_value((uint32_t)(floor >> 32));
    auto counts = [&](int id, float x) {
        return x > floor_value || (x == floor_value && row_key(x, id) >= floor);
    };
    auto bin_of = [&](float x) {  // of a token below the edge; grows as x falls
        const float d = (edge - x) * scale;
        return d < (float)(kBins - 1) ? (int)d : kBins - 1;
    };
    cl.sync();  // the shared arrays' earlier readers
    uint32_t* const limb = sh.bins[warp][0];
    for (int i = s.lane; i < 2 * kBins; i += 32) limb[i] = 0;
    if (t == 0) sh.n_cand = 0;
    __syncwarp();
    double top = 0.0;
    for_vectors_slow<DT>(row, s, ring, [&](int v, const uint4& u) {
        float x[N];
        decode<DT>(u, x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double w = counts(row.first(v) + j, x[j]) ? weight(x[j]) : 0.0;
            if (x[j] >= edge) {
                top += w;
            } else if (w > 0.0) {
                const int bin = bin_of(x[j]);
                // a whole number up to 2^40: its bits stand at the end of the sum's mantissa
                const double k = fma(w, per_unit, kBinMagic);
                const uint32_t lo = (uint32_t)__double2loint(k), hi = (uint32_t)__double2hiint(k);
                atomicAdd(&limb[bin], lo & 0xFFFFFu);
                atomicAdd(&limb[kBins + bin], __funnelshift_r(lo, hi, 20) & 0x1FFFFFu);
            }
        }
    });
    top = warp_sum(top);
    __syncthreads();
    // the CTA's bins, then the cluster's: thread t has two of them
    auto value = [&](const uint32_t* l, int bin) { return ((unsigned long long)l[kBins + bin] << 20) + l[bin]; };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        unsigned long long mine = 0;
        for (int w = 0; w < kRowWarps; ++w) mine += value(sh.bins[w][0], 2 * t + i);
        sh.bin_sum[2 * t + i] = mine;
    }
    all_gather(cl, sh.slots[1], g, top);
    cl.sync();
    unsigned long long all[2] = {0, 0};
    for (int i = 0; i < C; ++i) {
        const unsigned long long* from = cl.map_shared_rank(sh.bin_sum, i);
        all[0] += from[2 * t];
        all[1] += from[2 * t + 1];
    }
    const double tops = slots_sum(sh.slots[1], warps);
    unsigned long long incl = all[0] + all[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(~0u, incl, o);
        if (s.lane >= o) incl += y;
    }
    unsigned long long* const parts = reinterpret_cast<unsigned long long*>(sh.scan);
    if (s.lane == 31) parts[warp] = incl;
    if (t == 0) sh.sel_bin = kBins - 1;
    __syncthreads();
    unsigned long long before = 0, sum = 0;
    for (int i = 0; i < kRowWarps; ++i) {
        if (i < warp) before += parts[i];
        sum += parts[i];
    }
    incl += before;
    const double target = p * (tops + (double)sum * unit);
    const double need = (target - tops) * per_unit;
    if (!(need > 0.0)) return false;  // within the tops
    // one bin holds the border
    const unsigned long long mid = incl - all[1], low = mid - all[0];
    if ((double)low < need && (double)incl >= need) {
        const bool second = (double)mid < need;
        sh.sel_bin = (uint32_t)(2 * t + second);
        sh.bin_above = second ? mid : low;
    }
    __syncthreads();
    const int bin = (int)sh.sel_bin;
    if (bin == kBins - 1) return false;
    const double above = tops + (double)sh.bin_above * unit;
    // each warp's mass above the bin
    unsigned long long kept = 0;
    for (int i = s.lane; i < bin; i += 32) kept += value(limb, i);
    kept = warp_sum(kept);
    cl.sync();  // bins and sums are read; the list takes their place
    if (s.lane == 0) *cl.map_shared_rank(slots + g, 0) = top + (double)kept * unit;
    if (rank == 0 && t < warps) sh.bin_sum[t] = 0;
    append_slice<DT>(cl, sh, row, s,
                     [&](int id, float x) { return x < edge && bin_of(x) == bin && counts(id, x); });
    cl.sync();
    if (rank == 0) {
        int n = (int)sh.n_cand;
        bool ok = n > 0 && n <= kCand;
        if (ok) {
            const int per = (row.nv + warps - 1) / warps;
            double start = above;
            // a token that is kept goes to its warp's sum, in units
            auto keep = [&](unsigned long long key) {
                const double w = weight(key32_value((uint32_t)(key >> 32)));
                atomicAdd(&sh.bin_sum[(key_id(key) + row.shift) / N / per], (unsigned long long)(w * per_unit + 0.5));
            };
            if (n > kRowThreads) {
                // the bin once more in 256: sorting 1000 tokens takes 10 us, this 2
                uint32_t* const fine = reinterpret_cast<uint32_t*>(sh.w);  // two limbs
                unsigned long long* const part = reinterpret_cast<unsigned long long*>(fine + 512);
                constexpr uint32_t kPart = kCand - 256;  // what is left of sh.w
                auto fine_of = [&](unsigned long long key) {
                    const float d = (edge - key32_value((uint32_t)(key >> 32))) * scale - (float)bin;
                    return min(max((int)(d * 256.0f), 0), 255);
                };
                fine[t] = fine[256 + t] = 0;
                if (t == 0) sh.sel_above = 0;
                __syncthreads();
                for (int i = t; i < n; i += kRowThreads) {
                    const int f = fine_of(sh.cand[i]);
                    const double k = fma(weight(key32_value((uint32_t)(sh.cand[i] >> 32))), per_unit, kBinMagic);
                    const uint32_t lo = (uint32_t)__double2loint(k), hi = (uint32_t)__double2hiint(k);
                    atomicAdd(&fine[f], lo & 0xFFFFFu);
                    atomicAdd(&fine[256 + f], __funnelshift_r(lo, hi, 20) & 0x1FFFFFu);
                }
                __syncthreads();
                const unsigned long long mine = ((unsigned long long)fine[256 + t] << 20) + fine[t];
                unsigned long long sum = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long y = __shfl_up_sync(~0u, sum, o);
                    if (s.lane >= o) sum += y;
                }
                if (s.lane == 31) parts[warp] = sum;
                if (t == 0) {
                    sh.sel_bin = 255;
                    sh.bin_above = 0;
                }
                __syncthreads();
                for (int i = 0; i < warp; ++i) sum += parts[i];
                // (the last one in any case: rounding may leave the target past the end)
                const bool here = above + (double)(sum - mine) * unit < target &&
                                  (above + (double)sum * unit >= target || t == 255);
                if (here) {
                    sh.sel_bin = (uint32_t)t;
                    sh.bin_above = sum - mine;
                }
                __syncthreads();
                const int f = (int)sh.sel_bin;
                start = above + (double)sh.bin_above * unit;
                for (int i = t; i < n; i += kRowThreads) {
                    const int at = fine_of(sh.cand[i]);
                    if (at < f) keep(sh.cand[i]);
                    if (at != f) continue;
                    const uint32_t to = atomicAdd(&sh.sel_above, 1u);
                    if (to < kPart) part[to] = sh.cand[i];
                }
                __syncthreads();
                ok = sh.sel_above <= kPart;  // else one value's tokens nearly all
                n = ok ? (int)sh.sel_above : 0;
                for (int i = t; i < n; i += kRowThreads) sh.cand[i] = part[i];
                __syncthreads();
            }
            if (ok) {
                sort_candidates(sh.cand, n);
                for (int i = t; i < n; i += kRowThreads)
                    sh.w[i] = weight(key32_value((uint32_t)(sh.cand[i] >> 32)));
                __syncthreads();
                scan_weights(sh, n);
                int b = 0, e = n - 1;  // the token at which the target is reached
                while (b < e) {
                    const int m = (b + e) / 2;
                    if (start + sh.w[m] >= target) e = m;
                    else b = m + 1;
                }
                ok = start + (b > 0 ? sh.w[b - 1] : 0.0) + slack < target && start + sh.w[b] - slack >= target;
                for (int i = t; i <= b; i += kRowThreads) keep(sh.cand[i]);
                __syncthreads();
                if (t < warps) slots[t] += (double)sh.bin_sum[t] * unit;
                if (t < C) *cl.map_shared_rank(&sh.best, t) = sh.cand[b];
            }
        }
        if (t < C) *cl.map_shared_rank(&sh.verdict, t) = ok;
    }
    cl.sync();
    border = sh.best;
    return sh.verdict != 0;
}

}  // namespace qmm
