// speculative.cu -- which drafted tokens stand, and the token after them
// (ops.speculative_sample): the sampled form of a verify window.
//
// With p = softmax(l / T) of the model and q of the draft, position by
// position, token d_i stands while u_i q_i(d_i) < p_i(d_i).  At the first that
// does not, a token is drawn from max(p - q, 0); where the draft ends, from p.
// What comes out is distributed as the model alone would draw it.
//
// Two launches.  The first reads every row once, a cluster to a row: maximum
// and sum of weights (rows behind the end of a draft are not read).  The second
// is a cluster to a sequence: the tests, then the one draw from one or two
// rows.  Sums are fast ones with a bound; a test or a draw that the bound
// leaves open is made again with sums in 64 bits, so the tokens are those of
// 64-bit arithmetic.

#include "logits.cuh"

namespace qmm {

template <int DT>
QMM_DEVINL Row<DT> spec_row(const SpecArgs& a, long long b, int i) {  // i > n: the draft's row i - n - 1
    constexpr int bytes = Elem<DT>::kBytes;
    if (i <= a.n) return Row<DT>(static_cast<const char*>(a.logits) + b * a.stride_b * bytes, a.stride_i, i, a.V);
    return Row<DT>(static_cast<const char*>(a.draft) + b * a.dstride_b * bytes, a.dstride_i, i - a.n - 1, a.V);
}

QMM_DEVINL double spec_temperature(const SpecArgs& a, long long b, bool draft) {
    const float* rows = draft ? a.dt_rows : a.t_rows;
    return rows ? (double)rows[b] : draft ? a.dt : a.t;
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads, 4) spec_stats_kernel(const SpecArgs a) {
    __shared__ float tops[kMaxRowWarps];
    __shared__ double slots[kMaxRowWarps];
    __shared__ int args[kMaxRowWarps];
    cg::cluster_group cl = cg::this_cluster();
    cl.barrier_arrive();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), warps = C * kRowWarps;
    const int g = rank * kRowWarps + (threadIdx.x >> 5);
    const long long at = blockIdx.x / C;
    const long long b = at / (2 * a.n + 1);
    const int i = (int)(at % (2 * a.n + 1));
    const bool draft = i > a.n;
    // rows that come after the end of the draft are not looked at
    const int pos = draft ? i - a.n - 1 : i, need = draft ? pos + 1 : pos;
    bool skip = false;
    for (int j = 0; j < need; ++j) {
        const int64_t d = a.ids[b * a.n + j];
        skip |= d < 0 || d >= a.V;
    }
    if (skip) {
        cl.barrier_wait();
        return;
    }
    const Row<DT> row = spec_row<DT>(a, b, i);
    const Slice s = warp_slice<DT>(row, g, warps);
    const double T = spec_temperature(a, b, draft);
    const bool greedy = !(T > 0.0);
    const Scale c(greedy ? 1.0 : 1.0 / T);
    LaneSum acc;
    const float top = greedy ? stream_slice<DT, false>(row, s, c, acc) : stream_slice<DT, true>(row, s, c, acc);
    cl.barrier_wait();
    const float wtop = warp_max(top);
    all_gather(cl, tops, g, wtop);
    cl.sync();
    const float mx = slots_max(tops, warps);
    if (greedy) {
        int first = 0x7FFFFFFF;
        if (wtop == mx) {  // the warp's share again
            for_vectors_slow<DT>(row, s, [&](int v, const uint4& q) {
                float x[Elem<DT>::kVec];
                decode<DT>(q, x);
#pragma unroll
                for (int j = 0; j < Elem<DT>::kVec; ++j) {
                    const int id = row.first(v) + j;
                    if (x[j] == mx && id >= 0 && id < a.V) first = min(first, id);
                }
            });
        }
        all_gather(cl, args, g, __reduce_min_sync(~0u, first));
    } else {
        all_gather(cl, slots, g, warp_mass(acc, c, mx));
    }
    cl.sync();
    if (rank == 0 && threadIdx.x < 32) {
        RowStat st;
        st.mx = mx;
        st.arg = -1;
        st.sum = 1.0;
        if (greedy) {
            int first = 0x7FFFFFFF;
            for (int w = s.lane; w < warps; w += 32) first = min(first, args[w]);
            st.arg = __reduce_min_sync(~0u, first);
        } else {
            const double total = slots_sum(slots, warps);
            st.sum = c.fast(mx, T) && total >= 0.5 && total < CUDART_INF ? total : CUDART_NAN;
        }
        if (s.lane == 0) a.stats[at] = st;
    }
}

// One row's probabilities.
template <int DT>
struct Dist {
    Row<DT> row;
    RowStat st;
    bool greedy;
    Weight64 exact;

    QMM_DEVINL Dist(const SpecArgs& a, long long b, int i, const double* table)
        : row(spec_row<DT>(a, b, i)), st(a.stats[b * (2 * a.n + 1) + i]),
          greedy(!(spec_temperature(a, b, i > a.n) > 0.0)),
          exact(table, st.mx, greedy ? 1.0 : 1.0 / spec_temperature(a, b, i > a.n)) {
        if (dead()) st.sum = 1.0;
    }
    QMM_DEVINL double weight(int id, float x) const {
        if (dead()) return 0.0;
        if (greedy) return id == st.arg ? 1.0 : 0.0;
        return exact(x);
    }
    // against the sum at hand: exact weights, over a sum that may be a fast one
    QMM_DEVINL double prob(int id, float x) const { return weight(id, x) / st.sum; }
    QMM_DEVINL bool dead() const { return st.mx == -CUDART_INF_F; }  // masked throughout
};

// The row's sum in 64 bits, by the whole cluster.
template <int DT>
QMM_DEVINL void exact_sum(cg::cluster_group& cl, double* slots, Dist<DT>& d, int g, int warps) {
    if (d.greedy || d.dead()) return;
    double mass = 0.0;
    const Slice s = warp_slice<DT>(d.row, g, warps);
    for_vectors_slow<DT>(d.row, s, [&](int v, const uint4& q) {
        float x[Elem<DT>::kVec];
        decode<DT>(q, x);
#pragma unroll
        for (int j = 0; j < Elem<DT>::kVec; ++j) {
            const int id = d.row.first(v) + j;
            if (id >= 0 && id < d.row.V) mass += d.weight(id, x[j]);
        }
    });
    cl.sync();
    all_gather(cl, slots, g, warp_sum(mass));
    cl.sync();
    d.st.sum = slots_sum(slots, warps);
}

// Ids of a vector of p's row in q's row (whose start may lie otherwise).
template <int DT>
QMM_DEVINL void paired(const Row<DT>& p, const Row<DT>& q, int v, float (&y)[Elem<DT>::kVec]) {
    if (p.shift == q.shift) {
        decode<DT>(q.load(v), y);
        return;
    }
#pragma unroll
    for (int j = 0; j < Elem<DT>::kVec; ++j) {
        const int id = p.first(v) + j;
        y[j] = id >= 0 && id < q.V ? q.at(id) : -CUDART_INF_F;
    }
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads, 2) spec_decide_kernel(const SpecArgs a) {
    __shared__ double slots[kMaxRowWarps];
    __shared__ int sure_flag;
    __shared__ double table[32];
    fill_table(table);
    constexpr int N = Elem<DT>::kVec;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();  // every CTA is there before its memory is written
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), warps = C * kRowWarps;
    const int g = rank * kRowWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const long long b = blockIdx.x / C;
    const int64_t* ids = a.ids + b * a.n;
    const float* u = a.u + b * (a.n + 1);

    // the tests, 32 positions at a time, alike in every warp
    enum { kStands, kFails, kOpen, kEnds };
    int taken = 0;
    bool drafted = false;  // a drafted token fell
    for (bool more = true; more && taken < a.n;) {
        const int i = taken + lane;
        int state = kEnds;
        if (i < a.n) {
            const int64_t d = ids[i];
            if (d >= 0 && d < a.V) {
                bool before = true;  // rows past the draft's end have no sums
                for (int j = taken; j < i; ++j) before = before && ids[j] >= 0 && ids[j] < a.V;
                if (before) {
                    const Dist<DT> p(a, b, i, table), q(a, b, a.n + 1 + i, table);
                    const double wp = p.weight((int)d, p.row.at((int)d)), wq = q.weight((int)d, q.row.at((int)d));
                    const double left = (double)u[i] * wq / q.st.sum, right = wp / p.st.sum;
                    const double slack = (p.greedy && q.greedy ? 0.0 : 1.5 * kFastEps) * (left + right);
                    if (wp == 0.0) state = kFails;  // whatever the sums
                    else if (left + slack < right) state = kStands;
                    else if (left - slack >= right) state = kFails;
                    else state = kOpen;
                }
            }
        }
        const unsigned stop = __ballot_sync(~0u, state != kStands);
        const int at = stop ? __ffs(stop) - 1 : 32;
        taken += at;
        if (at == 32) continue;
        state = __shfl_sync(~0u, state, at);
        if (state == kOpen) {
            Dist<DT> p(a, b, taken, table), q(a, b, a.n + 1 + taken, table);
            exact_sum<DT>(cl, slots, p, g, warps);
            exact_sum<DT>(cl, slots, q, g, warps);
            const int d = (int)ids[taken];
            state = (double)u[taken] * q.prob(d, q.row.at(d)) < p.prob(d, p.row.at(d)) ? kStands : kFails;
        }
        if (state == kStands) {
            ++taken;
        } else {
            drafted = state == kFails;
            more = false;
        }
    }

    // the draw
    Dist<DT> p(a, b, taken, table);
    Dist<DT> q(a, b, drafted ? a.n + 1 + taken : taken, table);
    const Slice s = warp_slice<DT>(p.row, g, warps);
    const double draw = (double)u[a.n];
    int token = -1;
    bool mine = false;  // this lane writes the token
    // 0: fast sums; 1: sums in 64 bits; 2: nothing left of p - q, from p
    for (int tries = 0; tries < 3 && !p.dead(); ++tries) {
        const bool exact = tries > 0;
        const bool minus = drafted && tries < 2 && !q.dead();
        if (tries == 0 && !(p.st.sum > 0.0 && q.st.sum > 0.0)) continue;  // a sum is missing
        if (tries == 1) {
            exact_sum<DT>(cl, slots, p, g, warps);
            if (minus) exact_sum<DT>(cl, slots, q, g, warps);
        }
        double mass = 0.0;
        if (exact || p.greedy || q.greedy) {
            for_vectors_slow<DT>(p.row, s, [&](int v, const uint4& w) {
                float x[N], y[N];
                decode<DT>(w, x);
                if (minus) paired<DT>(p.row, q.row, v, y);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int id = p.row.first(v) + j;
                    if (id < 0 || id >= a.V) continue;
                    mass += minus ? fmax(p.prob(id, x[j]) - q.prob(id, y[j]), 0.0) : p.prob(id, x[j]);
                }
            });
        } else {
            const Scale cp(p.exact.inv_t), cq(q.exact.inv_t);
            const float ep = ceilf(p.st.mx * cp.c), eq = ceilf(q.st.mx * cq.c);
            const float fp = (float)(cp.against(ep, p.st.mx) / p.st.sum), fq = (float)(cq.against(eq, q.st.mx) / q.st.sum);
            for_vectors<DT>(p.row, s, [&](int v, const uint4& w) {
                float x[N], y[N];
                decode<DT>(w, x);
                if (minus) paired<DT>(p.row, q.row, v, y);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    x[j] = fp * ex2(fmaf(x[j], cp.c, -ep));
                    if (minus) x[j] = fmaxf(x[j] - fq * ex2(fmaf(y[j], cq.c, -eq)), 0.0f);
                }
                mass += (double)tree_sum<N>(x);
            });
        }
        cl.sync();
        all_gather(cl, slots, g, warp_sum(mass));
        cl.sync();
        const double total = slots_sum(slots, warps), target = draw * total;
        if (exact && minus && !(total > 0.0)) continue;
        // each of p and q is off by kFastEps of itself, in sums and in the target
        const double slack = exact || (p.greedy && (!minus || q.greedy)) ? 0.0 : 8.0 * kFastEps;
        const Place at = locate(slots, warps, target);
        bool sure = true;
        if (g == at.g) {
            const Found f = find_in_slice<DT>(p.row, s, at.base, target, [&](int id, float x) {
                const double w = p.prob(id, x);
                return minus ? fmax(w - q.prob(id, q.row.at(id)), 0.0) : w;
            });
            token = f.id;
            if (slack > 0.0) sure = f.id >= 0 && f.before + slack <= target && f.after - slack > target;
            mine = lane == 0;
            if (lane < C) *cl.map_shared_rank(&sure_flag, lane) = sure;
        } else if (at.g < 0 && g == 0) {
            if (lane < C) *cl.map_shared_rank(&sure_flag, lane) = exact;
            mine = lane == 0;
        }
        cl.sync();
        if (sure_flag) break;
        mine = false;
    }
    if (p.dead()) mine = g == 0 && lane == 0;  // nothing to draw from: -1
    if (mine) {
        int64_t* out = a.tokens + b * (a.n + 1);
        for (int i = 0; i <= a.n; ++i) out[i] = i < taken ? ids[i] : i == taken ? (int64_t)token : -1;
        a.accepted[b] = taken;
    }
}

}  // namespace qmm

namespace qmm_host {

size_t speculative_workspace(long long B, long long n) { return (size_t)(B * (2 * n + 1)) * sizeof(qmm::RowStat); }

template <int DT>
static int speculative_dt(const qmm::SpecArgs& a, cudaStream_t st) {
    const long long rows = (long long)a.B * (2 * a.n + 1);
    const int bytes = qmm::Elem<DT>::kBytes;
    const int rc = launch_rows(qmm::spec_stats_kernel<DT>, rows, row_cluster(rows, a.V, bytes), 0, st,
                               "speculative sums launch", a);
    if (rc) return rc;
    return launch_rows(qmm::spec_decide_kernel<DT>, a.B, row_cluster(a.B, a.V, bytes), 0, st, "speculative launch", a);
}

int launch_speculative(const qmm::SpecArgs& a, int dtype, cudaStream_t st) {
    if (dtype == QMM_BF16) return speculative_dt<0>(a, st);
    if (dtype == QMM_F16) return speculative_dt<1>(a, st);
    return speculative_dt<2>(a, st);
}

}  // namespace qmm_host
