// logits_select.cuh -- selection in a row of logits: a cluster's candidates
// for the largest tokens, and the border key of any count or mass.
#pragma once

#include "logits.cuh"

namespace qmm {

// A cluster's candidates are in its CTA 0.
struct SelectShared {
    union {
        float maxima[kRowThreads * kMaxCluster];  // one of each thread of the cluster (CTA 0's copy is used)
        double w[kCand];                          // the sorted candidates' weights
        uint32_t piv_count[2][kMaxRowWarps][8];
    };
    union {
        unsigned long long cand[kCand];  // CTA 0's copy is used
        double piv_mass[2][kMaxRowWarps][8];
    };
    double slots[2][kMaxRowWarps];
    float tops[kMaxRowWarps];
    uint32_t found[kMaxRowWarps];
    uint32_t hist[256];
    uint32_t n_cand, bound, sel_bin, sel_above;
    double scan[kRowWarps];
    unsigned long long best;
    int verdict;
};

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

// Candidates: every token with key32 >= bound, found again by the warps whose
// lanes' maxima reach it (lane `owner` holds the slice's vectors owner, owner +
// 32, ..).  They go to CTA 0's list in any order; returns how many this warp
// found.  The list's own count may pass kCand; no more than that are written.
template <int DT>
QMM_DEVINL uint32_t push_candidates(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s,
                                    float top, uint32_t bound) {
    constexpr int N = Elem<DT>::kVec;
    unsigned owners = __ballot_sync(~0u, key32(top) >= bound && s.begin + s.lane < s.end);
    uint32_t* count = cl.map_shared_rank(&sh.n_cand, 0);
    unsigned long long* list = cl.map_shared_rank(sh.cand, 0);
    uint32_t found = 0;
    while (owners) {
        const int owner = __ffs(owners) - 1;
        owners &= owners - 1;
        for (int v = s.begin + owner + 32 * s.lane; v < s.end; v += 32 * 32) {
            float x[N];
            decode<DT>(row.load(v), x);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int id = row.first(v) + j;
                if (id < 0 || id >= row.V || key32(x[j]) < bound) continue;
                ++found;
                const uint32_t at = atomicAdd(count, 1u);
                if (at < kCand) list[at] = row_key(x[j], id);
            }
        }
    }
    return warp_sum(found);
}

// Descending bitonic sort of the first n candidates in place (padded with 0,
// which no token's key is).  One CTA.
QMM_DEVINL void sort_candidates(unsigned long long* k, int n) {
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

// The border key: the largest key b in [lo, hi) such that the tokens with keys
// >= b reach `target` (their number, or with MASS the sum of their weights in
// 64 bits); lo if all of them do not.  All warps of the cluster; the rounds cut
// the range into eight and end when one token is left in it, 22 rounds at most.
template <int DT, bool MASS>
QMM_DEVINL unsigned long long border_key(cg::cluster_group& cl, SelectShared& sh, const Row<DT>& row, const Slice& s,
                                         int g, int warps, float mx, double inv_t, unsigned long long lo,
                                         unsigned long long hi, double target) {
    constexpr int N = Elem<DT>::kVec;
    uint32_t in_lo = 0xFFFFFFFFu, in_hi = 0;
    cl.sync();  // the shared arrays' earlier readers
    for (int round = 0; hi - lo > 1 && in_lo - in_hi > 1; ++round) {
        const unsigned long long step = (hi - lo) / 8 > 0 ? (hi - lo) / 8 : 1;
        // pivots lo + j step, j = 0 .. 7, below hi
        uint32_t n[8];
        double m[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            n[j] = 0;
            m[j] = 0.0;
        }
        for_vectors<DT>(row, s, [&](int v, const uint4& u) {
            float x[N];
            decode<DT>(u, x);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int id = row.first(v) + e;
                if (id < 0 || id >= row.V) continue;
                const unsigned long long k = row_key(x[e], id);
                if (k < lo) continue;
                const double w = MASS ? weight64(x[e], mx, inv_t) : 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (k >= lo + j * step) {
                        ++n[j];
                        if (MASS) m[j] += w;
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
        // lane j < 8 of every warp: pivot j's totals, in the order of warps
        uint32_t tn = 0;
        double tm = 0.0;
        if (s.lane < 8) {
            for (int i = 0; i < warps; ++i) {
                tn += sh.piv_count[buf][i][s.lane];
                if (MASS) tm += sh.piv_mass[buf][i][s.lane];
            }
        }
        const bool reach = s.lane < 8 && lo + s.lane * step < hi && (MASS ? tm : (double)tn) >= target;
        const unsigned reached = __ballot_sync(~0u, reach);
        if (!(reached & 1u)) return lo;  // not even all of them: first round only
        const int at = 31 - __clz(reached);
        in_lo = __shfl_sync(~0u, tn, at);
        const unsigned long long base = lo;
        lo = base + at * step;
        if (at < 7 && base + (at + 1) * step < hi) {
            hi = base + (at + 1) * step;
            in_hi = __shfl_sync(~0u, tn, at + 1);
        }
    }
    return lo;
}

}  // namespace qmm
