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
//
// The first launch is bound by memory and the exponential unit (both near 65%),
// the second by its chain: tests, a pass over two rows in L2, the exchange, the
// place.  B200, V 248320: one sequence of 4 drafted tokens 24 us, 48 of up to 3
// 117 to 147 us (44 and the draws; a sequence whose draw is made again takes 90
// of these).  Where the model's rows and the draft's start differently, as with
// an odd V, the draft's are read element by element: 201 us at V 248321.

#include "logits.cuh"
#include "tma.cuh"

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
    __shared__ WarpStat stats[kMaxRowWarps];
    __shared__ int args[kMaxRowWarps];
    cg::cluster_group cl = cg::this_cluster();
    cl.barrier_arrive();
    pdl_launch_dependents();  // the second kernel's start beside this one's end
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), warps = C * kRowWarps;
    const int g = rank * kRowWarps + (threadIdx.x >> 5);
    const long long at = blockIdx.x / C;
    const long long b = at / (2 * a.n + 1);
    const int i = (int)(at % (2 * a.n + 1));
    const bool draft = i > a.n;
    // rows that come after the end of the draft are not looked at
    const int pos = draft ? i - a.n - 1 : i, need = draft ? pos + 1 : pos;
    bool skip = false;
    for (int j = threadIdx.x & 31; j < need; j += 32) {
        const int64_t d = a.ids[b * a.n + j];
        skip |= d < 0 || d >= a.V;
    }
    if (__any_sync(~0u, skip)) {
        cl.barrier_wait();
        return;
    }
    const Row<DT> row = spec_row<DT>(a, b, i);
    const Slice s = warp_slice<DT>(row, g, warps);
    const double T = spec_temperature(a, b, draft);
    const bool greedy = !(T > 0.0);
    const Scale c(greedy ? 1.0 : 1.0 / T);
    LaneSum acc;
    const float top = greedy ? stream_slice<DT, false, false>(row, s, c, acc).first
                             : stream_slice<DT, true, false>(row, s, c, acc).first;
    const WarpStat stat = warp_stat(top, acc);
    cl.barrier_wait();
    all_gather(cl, stats, g, stat);
    cl.sync();
    float mx;
    double total;
    row_stat(stats, warps, c, mx, total, nullptr);
    if (greedy) {
        int first = 0x7FFFFFFF;
        if (stat.top == mx) {  // the warp's share again
            for_vectors_rare<DT>(row, s, [&](int v, const uint4& q) {
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
        cl.sync();
    }
    if (rank == 0 && threadIdx.x < 32) {
        RowStat st;
        st.mx = mx;
        st.arg = -1;
        st.sum = 1.0;
        st.inv_t = greedy ? 1.0 : 1.0 / T;
        if (greedy) {
            int first = 0x7FFFFFFF;
            for (int w = s.lane; w < warps; w += 32) first = min(first, args[w]);
            st.arg = __reduce_min_sync(~0u, first);
        } else {
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
        : Dist(a, b, i, table, spec_temperature(a, b, i > a.n)) {}
    QMM_DEVINL Dist(const SpecArgs& a, long long b, int i, const double* table, double T)
        : row(spec_row<DT>(a, b, i)), st(a.stats[b * (2 * a.n + 1) + i]), greedy(!(T > 0.0)),
          exact(table, st.mx, T, st.inv_t) {
        if (dead()) st.sum = 1.0;
    }
    QMM_DEVINL double weight(int id, float x) const {
        if (dead()) return 0.0;
        if (greedy) return id == st.arg ? 1.0 : 0.0;
        return exact(x);
    }
    // against the sum at hand: exact weights, over a sum that may be a fast one
    QMM_DEVINL double prob(int id, float x) const { return weight(id, x) / st.sum; }
    // a vector's, whose element 0 is token `first`
    QMM_DEVINL void probs(int first, const float (&x)[Elem<DT>::kVec], double (&w)[Elem<DT>::kVec]) const {
        const double part = dead() ? 0.0 : 1.0 / st.sum;
        if (greedy) {
#pragma unroll
            for (int j = 0; j < Elem<DT>::kVec; ++j) w[j] = first + j == st.arg ? part : 0.0;
        } else {
#pragma unroll
            for (int j = 0; j < Elem<DT>::kVec; ++j) w[j] = exact(x[j]) * part;
        }
    }
    QMM_DEVINL bool dead() const { return st.mx == -CUDART_INF_F; }  // masked throughout
};

// Ids of a vector of p's row in q's row, whose start may lie otherwise.
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

// f(vector index, p's elements, q's) over the warp's slice of p's row; q's are
// read where BOTH, with the next vectors of either on their way (q's row lies
// alike: its vectors are whole where p's are).
template <int DT, typename F>
QMM_DEVINL void for_pairs(const Row<DT>& p, const Row<DT>& q, const Slice& s, Ring ring, bool both, F&& f) {
    constexpr int N = Elem<DT>::kVec;
    if (!both || p.shift != q.shift) {
        for_vectors_slow<DT>(p, s, ring, [&](int v, const uint4& u) {
            float x[N], y[N];
            decode<DT>(u, x);
            if (both) paired<DT>(p, q, v, y);
            f(v, x, y);
        });
        return;
    }
    const int t = threadIdx.x;
    int v = s.begin + s.lane;
    constexpr int kAhead = kRing / 2 - 1;  // pairs
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        if (v + 32 * i < s.end) {
            async_copy16(&ring[2 * i][t], p.base + 16LL * (v + 32 * i));
            async_copy16(&ring[2 * i + 1][t], q.base + 16LL * (v + 32 * i));
        }
        async_commit();
    }
    auto ends = [&](int at) {
        float x[N], y[N];
        decode<DT>(p.load(at), x);
        decode<DT>(q.load(at), y);
        f(at, x, y);
    };
    if (s.lane == 0 && s.head >= 0) ends(s.head);
    int slot = 0;
#pragma unroll 1
    for (; v < s.end; v += 32) {
        async_wait<kAhead - 1>();
        float x[N], y[N];
        decode<DT>(ring[2 * slot][t], x);
        decode<DT>(ring[2 * slot + 1][t], y);
        const int free = slot == 0 ? kAhead : slot - 1, ahead = v + 32 * kAhead;
        if (ahead < s.end) {
            async_copy16(&ring[2 * free][t], p.base + 16LL * ahead);
            async_copy16(&ring[2 * free + 1][t], q.base + 16LL * ahead);
        }
        async_commit();
        slot = slot == kAhead ? 0 : slot + 1;
        f(v, x, y);
    }
    async_wait<0>();
    if (s.lane == 0 && s.tail >= 0) ends(s.tail);
}

// The sums of both rows (both false: of p's) in 64 bits, by the whole cluster.
struct TwoSums {
    double p, q;
};

// Not inlined: it hardly runs, and what a call does run stays short.
template <int DT>
__device__ __noinline__ void exact_sums(cg::cluster_group& cl, TwoSums* slots, Ring ring, Dist<DT>& p, Dist<DT>& q, int g,
                                        int warps, bool both) {
    constexpr int N = Elem<DT>::kVec;
    TwoSums mass{0.0, 0.0};
    const Slice s = warp_slice<DT>(p.row, g, warps);
    const Weight64 wp = p.exact, wq = q.exact;  // in registers
    for_pairs<DT>(p.row, q.row, s, ring, both, [&](int, const float (&x)[N], const float (&y)[N]) {
        double w[N];  // past the ends -infinity: nothing
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = wp(x[j]);
        mass.p += tree_sum(w);
        if (!both) return;
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = wq(y[j]);
        mass.q += tree_sum(w);
    });
    mass.p = warp_sum(mass.p);
    mass.q = warp_sum(mass.q);
    cl.sync();
    all_gather(cl, slots, g, mass);
    cl.sync();
    double sp = 0.0, sq = 0.0;
    for (int i = s.lane; i < warps; i += 32) {
        sp += slots[i].p;
        sq += slots[i].q;
    }
    sp = warp_sum(sp);
    sq = warp_sum(sq);
    if (!p.greedy && !p.dead()) p.st.sum = sp;
    if (both && !q.greedy && !q.dead()) q.st.sum = sq;
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads, 2) spec_decide_kernel(const SpecArgs a) {
    __shared__ double slots[2][kMaxRowWarps];
    __shared__ TwoSums sums[kMaxRowWarps];
    __shared__ int sure_flag;
    __shared__ FindShared find;
    __shared__ double table[32];
    __shared__ uint4 ring_memory[kRing][kRowThreads];
    const Ring ring = ring_memory;
    fill_table(table);
    constexpr int N = Elem<DT>::kVec;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();  // every CTA is there before its memory is written
    pdl_wait();  // the sums; nothing of global memory is read before
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
            exact_sums<DT>(cl, sums, ring, p, q, g, warps, true);
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
    bool mine = false;  // this thread writes the token
    // 0: fast sums; 1: sums in 64 bits; 2: nothing left of p - q, from p
    for (int tries = 0; tries < 3 && !p.dead(); ++tries) {
        const bool exact = tries > 0;
        const bool minus = drafted && tries < 2 && !q.dead();
        if (tries == 0 && !(p.st.sum > 0.0 && q.st.sum > 0.0)) continue;  // a sum is missing
        if (tries == 1) {
            exact_sums<DT>(cl, sums, ring, p, q, g, warps, minus);
        }
        auto weigh = [&](int v, const float (&x)[N], const float (&y)[N], double (&out)[N]) {
            double other[N];
            const int first = p.row.first(v);
            p.probs(first, x, out);
            if (minus) q.probs(first, y, other);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (minus) out[j] = fmax(out[j] - other[j], 0.0);
                if (first + j < 0 || first + j >= a.V) out[j] = 0.0;
            }
        };
        double mass = 0.0;
        if (exact || p.greedy || q.greedy) {
            for_pairs<DT>(p.row, q.row, s, ring, minus, [&](int v, const float (&x)[N], const float (&y)[N]) {
                double out[N];
                weigh(v, x, y, out);
                mass += tree_sum(out);
            });
        } else {
            const Scale cp(p.exact.inv_t), cq(q.exact.inv_t);
            const float ep = ceilf(p.st.mx * cp.c), eq = ceilf(q.st.mx * cq.c);
            const float fp = (float)(cp.against(ep, p.st.mx) / p.st.sum), fq = (float)(cq.against(eq, q.st.mx) / q.st.sum);
            for_pairs<DT>(p.row, q.row, s, ring, minus, [&](int v, const float (&x)[N], const float (&y)[N]) {
                float w[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    w[j] = fp * ex2(fmaf(x[j], cp.c, -ep));
                    if (minus) w[j] = fmaxf(w[j] - fq * ex2(fmaf(y[j], cq.c, -eq)), 0.0f);
                }
                mass += (double)tree_sum(w);
            });
        }
        double* const places = slots[tries & 1];
        all_gather(cl, places, g, warp_sum(mass));
        cl.sync();
        const double total = slots_sum(places, warps), target = draw * total;
        if (exact && minus && !(total > 0.0)) continue;
        // each of p and q is off by kFastEps of itself, in sums and in the target
        const double slack = exact || (p.greedy && (!minus || q.greedy)) ? 0.0 : 8.0 * kFastEps;
        const Place at = locate(places, warps, target);
        if (at.g >= 0 && rank == at.g / kRowWarps) {
            const Found f =
                find_in_slice<DT>(p.row, warp_slice<DT>(p.row, at.g, warps), at.base, target, ring, find,
                                              [&](int v, const uint4& w, double (&out)[N]) {
                                                  float x[N], y[N];
                                                  decode<DT>(w, x);
                                                  if (minus) paired<DT>(p.row, q.row, v, y);
                                                  weigh(v, x, y, out);
                                              });
            token = f.id;
            const bool sure = slack == 0.0 || (f.id >= 0 && f.before + slack <= target && f.after - slack > target);
            if (threadIdx.x < C) *cl.map_shared_rank(&sure_flag, threadIdx.x) = sure;
            mine = threadIdx.x == 0;
        } else if (at.g < 0 && rank == 0) {
            if (threadIdx.x < C) *cl.map_shared_rank(&sure_flag, threadIdx.x) = exact;
            mine = threadIdx.x == 0;
        }
        cl.sync();
        if (sure_flag) break;
        mine = false;
    }
    if (p.dead()) mine = rank == 0 && threadIdx.x == 0;  // nothing to draw from: -1
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
    const int rc = launch_rows(qmm::spec_stats_kernel<DT>, qmm::kRowThreads, rows,
                               row_cluster(rows, a.V, bytes, 4 * 148, 128), 0, st, "speculative sums launch", a);
    if (rc) return rc;
    return launch_rows<true>(qmm::spec_decide_kernel<DT>, qmm::kRowThreads, a.B, row_cluster(a.B, a.V, bytes, 4 * 148),
                             0, st, "speculative launch", a);
}

int launch_speculative(const qmm::SpecArgs& a, int dtype, cudaStream_t st) {
    if (dtype == QMM_BF16) return speculative_dt<0>(a, st);
    if (dtype == QMM_F16) return speculative_dt<1>(a, st);
    return speculative_dt<2>(a, st);
}

}  // namespace qmm_host
