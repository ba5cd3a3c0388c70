// sample.cu -- a token a row from a given uniform number: temperature, top-k,
// top-p, min-p (ops.sample).
//
// With w_i = exp((l_i - max) / T) and the tokens in the order of (logit
// descending, id ascending), kept are the first top_k; of these, as long as
// the mass before a token is below top_p times theirs; and those with
// w_i >= min_p.  The answer is the first id, in the order of ids, at which the
// kept weights add up to more than u times their sum.  Every kept set is a
// prefix of the order, so it is {key >= border} for one 64-bit key.
//
// The ids are those of 64-bit arithmetic.  Where sums over the whole row are
// needed (top-p without top-k, no filter at all) a 32-bit pass gives them with
// a bound on their error; only a row whose decision lies within that bound of
// a border takes a second pass in 64 bits.
//
// One reading of memory bounds it from below, and a chain of steps beside that:
// a row's cluster reads (2 us of the 12 of a single row of 248320), exchanges
// maxima, collects the candidates, and CTA 0 sorts and draws.  With top-k no
// exponential is taken but of the candidates.  Measured on a B200, V 248320: one
// row, top-k 20 and top-p 0.95, 12 us; 65 rows of 50021 with settings of their
// own 17 us; 128 rows with top-p 0.95, half of them open, 160 to 178 us (floor
// 9.7: no unit is busy, the 64-bit pipe at 5%; a cluster's other CTAs wait at
// barriers for the one that lists and sorts); 512 rows of fp32 without a filter
// 180 us (floor 78: 129 where the model is sure, the rest second passes).

#include "logits_select.cuh"

namespace qmm {

// What CTA 0 makes of the candidates: the answer; a sum in 64 bits is needed;
// the border, but more kept tokens than it draws from itself; not enough of them.
enum { kDone, kNeedSum, kBorder, kGeneral };
constexpr int kDrawHere = 2 * kRowThreads;
static_assert(kDrawHere <= kBins, "their weights lie in bin_sum");
// What a row with top-p alone lists first: enough where the model is sure of
// itself, and about 180 tokens, which a CTA sorts in one turn.
constexpr int kNucleus = 128;

// How many of the first n running sums stand before `limit`: the tokens whose
// mass before them (the sum of the one above) is below it.  The first always is.
QMM_DEVINL int count_before(const double* sums, int n, double limit) {
    int lo = 1, hi = n;  // the first i >= 1 with sums[i - 1] >= limit
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sums[mid - 1] >= limit) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// FILTERS false: no row has a filter or is greedy, by the call's numbers.  That
// kernel does without the selection's memory and registers: a fourth CTA to an SM.
template <int DT, bool FILTERS>
__global__ void __launch_bounds__(kRowThreads, FILTERS ? 3 : 4) sample_kernel(const SampleArgs a) {
    extern __shared__ uint4 memory[];
    SelectShared& sh = *reinterpret_cast<SelectShared*>(memory + kRing * kRowThreads);
    const Ring ring = reinterpret_cast<Ring>(memory);
    cg::cluster_group cl = cg::this_cluster();
    cl.barrier_arrive();  // waited for before the first access to another CTA
    if (FILTERS && threadIdx.x == 0) sh.n_cand = 0;
    fill_table(sh.table);
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), warps = C * kRowWarps;
    const int g = rank * kRowWarps + (threadIdx.x >> 5);
    const long long r = blockIdx.x / C;
    const Row<DT> row(a.logits, a.stride, r, a.V);
    const Slice s = warp_slice<DT>(row, g, warps);

    double T = a.t_rows ? (double)a.t_rows[r] : a.t;
    int k = FILTERS && a.k_rows ? a.k_rows[r] : a.k;
    const double p = FILTERS && a.p_rows ? (double)a.p_rows[r] : a.p;
    double mp = FILTERS && a.m_rows ? (double)a.m_rows[r] : a.m;
    if (!(T > 0.0)) {  // greedy
        T = 1.0;
        k = 1;
    }
    const bool k_on = FILTERS && k >= 1 && k < a.V, p_on = FILTERS && p < 1.0 && !(k_on && k == 1);
    const bool m_on = FILTERS && mp > 1e-300 && !(k_on && k == 1);  // no weight is below that
    if (mp > 1.0) mp = 1.0;
    const double inv_t = 1.0 / T, u = (double)a.u[r];
    const bool sum = !k_on && (p_on || !m_on);
    const Scale c(inv_t);

    // one pass over memory
    LaneSum acc;
    const LaneTop top =
        sum ? stream_slice<DT, true, FILTERS>(row, s, c, acc) : stream_slice<DT, false, true>(row, s, c, acc);
    const WarpStat stat = warp_stat(top.first, acc, sum);
    const bool select = k_on || p_on;  // a bound from maxima
    const int want = k_on ? k : kNucleus;
    const int lanes = lanes_to_group(warps, want);
    // Beyond, the bins: 16 rows of 248320, k 1000, on 16 CTAs each, listed 60 us, by bins 123; 300 rows of 50000
    // on 8 CTAs for the list's sake 323, by bins on 2 CTAs 199.
    const bool listed = select ? 2 * want <= C * kRowThreads || want <= kRowThreads : m_on;
    cl.barrier_wait();
    all_gather(cl, sh.stats, g, stat);
    if (select && listed) publish_maxima(cl, sh, g, lanes, top.first);
    cl.sync();
    float mx;
    double total;
    row_stat(sh.stats, warps, c, mx, total, sh.slots[0], sum);
    if (mx == -CUDART_INF_F) {  // nothing to draw from
        if (rank == 0 && threadIdx.x == 0) a.ids[r] = -1;
        return;
    }
    const bool fast = sum && c.fast(mx, T) && total >= 0.5 && total < CUDART_INF;  // else 64 bits
    const Weight64 weight(sh.table, mx, T, inv_t);

    // smallest key that min-p keeps; masked tokens have none
    uint32_t kmin = kKeyNegInf + 1;
    if (m_on) {
        const float guess = (float)((double)mx + T * log(mp));
        kmin = lowest_kept(kmin, key32(mx), key32(guess), [&](uint32_t b) { return weight(key32_value(b)) >= mp; });
    }
    // Top-k without top-p: tokens below min-p play no part.
    uint32_t bound = kmin;
    if (select && listed) {
        const uint32_t b = kth_bound(sh, warps * (32 / lanes), want);
        bound = max(b, kKeyNegInf + 1);
        if (!(k_on && p_on)) bound = max(bound, kmin);
    }
    unsigned long long border = (unsigned long long)kmin << 32;
    bool bordered = false;

    if (listed) {
        const uint32_t mine = push_candidates<DT>(cl, sh, row, s, top, bound);
        all_gather(cl, sh.found, g, mine);
        cl.sync();
        uint32_t n = 0;
        for (int i = s.lane; i < warps; i += 32) n += sh.found[i];
        n = warp_sum(n);
        if (n <= kCand) {
            // one CTA's work; the others wait only where it may end otherwise
            const bool sure = k_on && k <= kRowThreads;
            if (rank != 0 && sure) return;
            bool sorted = false;
            double eps = k_on ? 0.0 : fast ? kFastEps : 1.0;
            // Of the tokens that are drawn from: a difference of the running sums in sh.w would be 0 for one below
            // 2^-53 of them, which u = 0 may ask for.
            double* const own = reinterpret_cast<double*>(sh.bin_sum);
            for (;;) {
                if (rank == 0) {
                    int verdict = kDone;
                    if (!k_on && p_on && bound > kmin && eps < 1.0 && !sorted) {
                        // an open row: the list is far from top_p, and is not worth its sorting
                        double listed_mass = 0.0;
                        for (int i = threadIdx.x; i < (int)n; i += kRowThreads)
                            listed_mass += weight(key32_value((uint32_t)(sh.cand[i] >> 32)));
                        if (cta_sum(sh, listed_mass) < p * total * (1.0 - 2.0 * eps)) verdict = kGeneral;
                    }
                    int kept = (int)n;
                    if (verdict == kDone && !sorted) {
                        sort_candidates(sh.cand, (int)n);
                        for (int i = threadIdx.x; i < (int)n; i += kRowThreads) {
                            const double w = weight(key32_value((uint32_t)(sh.cand[i] >> 32)));
                            sh.w[i] = w;
                            if (i < kDrawHere) own[i] = w;
                        }
                        __syncthreads();
                        scan_weights(sh, (int)n);
                        sorted = true;
                    }
                    if (k_on && k < kept) kept = k;
                    if (p_on && verdict == kDone) {
                        const double all = k_on ? sh.w[kept - 1] : total;
                        const int lo = count_before(sh.w, kept, p * all * (1.0 - eps));
                        const int hi = count_before(sh.w, kept, p * all * (1.0 + eps));
                        const bool open = !k_on && bound > kmin && !(sh.w[kept - 1] >= p * all * (1.0 + eps));
                        if (eps == 1.0) verdict = kNeedSum;
                        else if (open) verdict = eps > 0.0 && sh.w[kept - 1] >= p * all * (1.0 - eps) ? kNeedSum : kGeneral;
                        else if (lo != hi) verdict = kNeedSum;
                        kept = hi;
                    }
                    // of them, those that min-p keeps
                    int lo = 0, hi = kept;
                    while (lo < hi) {
                        const int mid = (lo + hi) / 2;
                        if ((uint32_t)(sh.cand[mid] >> 32) >= kmin) lo = mid + 1;
                        else hi = mid;
                    }
                    kept = lo;
                    if (verdict == kDone && kept > kDrawHere) verdict = kBorder;
                    if (verdict == kDone) {
                        // the first id at which the sum over kept tokens with ids up to it passes u W
                        const double target = u * sh.w[kept - 1];
                        if (threadIdx.x == 0) sh.best = ~0ull;
                        __syncthreads();
                        unsigned long long best = ~0ull;
                        for (int j = threadIdx.x; j < kept; j += kRowThreads) {
                            const int id = key_id(sh.cand[j]);
                            double run = 0.0;
                            for (int i = 0; i < kept; ++i)
                                if (key_id(sh.cand[i]) <= id) run += own[i];
                            if (own[j] > 0.0) {
                                // past the target: the smallest id; if none is, the largest id of all
                                const unsigned long long code =
                                    run > target ? (unsigned long long)id : (1ull << 40) + (0xFFFFFFFFu - (uint32_t)id);
                                best = code < best ? code : best;
                            }
                        }
                        atomicMin(&sh.best, best);
                        __syncthreads();
                        if (threadIdx.x == 0) {
                            const unsigned long long b = sh.best;
                            a.ids[r] = b < (1ull << 40) ? (int64_t)b : (int64_t)(0xFFFFFFFFu - (uint32_t)(b - (1ull << 40)));
                        }
                    }
                    if (!sure && threadIdx.x < C) {
                        *cl.map_shared_rank(&sh.verdict, threadIdx.x) = verdict;
                        if (verdict == kBorder) *cl.map_shared_rank(&sh.best, threadIdx.x) = sh.cand[kept - 1];
                    }
                }
                if (sure) return;
                cl.sync();
                const int verdict = sh.verdict;
                if (verdict == kDone) return;
                if (verdict == kBorder) border = sh.best;
                if (verdict != kNeedSum) {
                    bordered = verdict == kBorder;
                    break;
                }
                // the row's sum in 64 bits, then again
                double mass = 0.0;
                for_vectors_slow<DT>(row, s, ring, [&](int v, const uint4& q) {
                    float x[Elem<DT>::kVec];
                    double w[Elem<DT>::kVec];
                    decode<DT>(q, x);
#pragma unroll
                    for (int j = 0; j < Elem<DT>::kVec; ++j) w[j] = weight(x[j]);
                    mass += tree_sum(w);
                });
                all_gather(cl, sh.slots[1], g, warp_sum(mass));
                cl.sync();
                total = slots_sum(sh.slots[1], warps);
                eps = 0.0;
            }
        }
    }

    if (!select && !m_on && fast) {  // no filter: the warps' fast masses are the distribution
        __syncthreads();
        const double target = u * total, slack = 2.0 * kFastEps * total;
        const Place at = locate(sh.slots[0], warps, target);
        if (rank == at.g / kRowWarps) {
            const Found f = find_in_slice<DT>(row, warp_slice<DT>(row, at.g, warps), at.base, target, ring, sh.find,
                                              [&](int, const uint4& q, double (&w)[Elem<DT>::kVec]) {
                float x[Elem<DT>::kVec];
                decode<DT>(q, x);
#pragma unroll
                for (int j = 0; j < Elem<DT>::kVec; ++j) w[j] = weight(x[j]);
            });
            const bool sure = f.id >= 0 && f.before + slack <= target && f.after - slack > target;
            if (sure && threadIdx.x == 0) a.ids[r] = f.id;
            if (threadIdx.x < C) *cl.map_shared_rank(&sh.verdict, threadIdx.x) = sure ? kDone : kGeneral;
        }
        cl.sync();
        if (sh.verdict == kDone) return;
    }

    // the general way: borders by bins or search, masses and place in 64 bits
    const int per = (row.nv + warps - 1) / warps;
    const unsigned long long bottom = (unsigned long long)(kKeyNegInf + 1) << 32;
    unsigned long long from = bottom;
    if (k_on && !bordered) {
        float low = CUDART_INF_F;
        for (int i = s.lane; i < warps; i += 32) low = fminf(low, sh.stats[i].e);
        low = -warp_max(-low);
        if (!kth_by_bins<DT>(cl, sh, row, s, mx, low, k, from))
            from = border_key<DT, false>(cl, sh, row, s, g, warps, ring, weight, bottom, (double)k);
    }
    if (p_on && !bordered && per * Elem<DT>::kVec <= kBinTokens) {
        // without top-k down to where what is left, V tokens at most, is half of what top-p leaves out
        const float edge = k_on ? mx : key32_value(bound);
        const double deep = k_on ? ((double)mx - (double)key32_value((uint32_t)(from >> 32))) * inv_t * 1.001
                                 : log(2.0 * row.V * weight(edge) / ((1.0 - p) * total));
        unsigned long long found;
        double slack;
        if (border_by_bins<DT>(cl, sh, row, s, g, warps, ring, weight, p, edge, deep, from, k_on ? k : row.V,
                               sh.slots[0], found, slack)) {
            from = found;
            if (from >= border) {  // min-p keeps them all: CTA 0 has each warp's mass
                if (rank != 0) return;
                const uint32_t from32 = (uint32_t)(from >> 32);
                auto from_on = [&](int v, const uint4& q, double (&w)[Elem<DT>::kVec]) {
                    float x[Elem<DT>::kVec];
                    decode<DT>(q, x);
#pragma unroll
                    for (int j = 0; j < Elem<DT>::kVec; ++j) {
                        const uint32_t k32 = key32(x[j]);
                        const bool out = k32 < from32 || (k32 == from32 && row_key(x[j], row.first(v) + j) < from);
                        w[j] = out ? 0.0 : weight(x[j]);
                    }
                };
#pragma unroll 1
                for (;; slack = 0.0) {
                    const double target = u * slots_sum(sh.slots[0], warps);
                    const Place at = locate(sh.slots[0], warps, target);
                    const Found f = find_in_slice<DT>(row, warp_slice<DT>(row, at.g, warps), at.base, target, ring,
                                                      sh.find, from_on);
                    if (slack == 0.0 || (f.id >= 0 && f.before + slack <= target && f.after - slack > target)) {
                        if (threadIdx.x == 0) a.ids[r] = f.id;
                        return;
                    }
                    // the masses in 64 bits, by this CTA alone: the others have left
                    for (int i = threadIdx.x >> 5; i < warps; i += kRowWarps) {
                        double mass = 0.0;
                        for_vectors_slow<DT>(row, warp_slice<DT>(row, i, warps), ring, [&](int v, const uint4& q) {
                            double w[Elem<DT>::kVec];
                            from_on(v, q, w);
                            mass += tree_sum(w);
                        });
                        mass = warp_sum(mass);
                        if (s.lane == 0) sh.slots[0][i] = mass;
                    }
                    __syncthreads();
                }
            }
            bordered = true;
        }
    }
    if (select && !bordered) {
        if (p_on) from = border_key<DT, true>(cl, sh, row, s, g, warps, ring, weight, from, p);
        if (from > border) border = from;
    }
    const uint32_t border32 = (uint32_t)(border >> 32);
    auto kept = [&](int v, const uint4& q, double (&w)[Elem<DT>::kVec]) {
        float x[Elem<DT>::kVec];
        decode<DT>(q, x);
#pragma unroll
        for (int j = 0; j < Elem<DT>::kVec; ++j) {  // -infinity past the ends
            const uint32_t k32 = key32(x[j]);
            w[j] = k32 < border32 || (k32 == border32 && row_key(x[j], row.first(v) + j) < border) ? 0.0 : weight(x[j]);
        }
    };
    double mass = 0.0;
    for_vectors_slow<DT>(row, s, ring, [&](int v, const uint4& q) {
        double w[Elem<DT>::kVec];
        kept(v, q, w);
        mass += tree_sum(w);
    });
    cl.sync();
    all_gather(cl, sh.slots[0], g, warp_sum(mass));
    cl.sync();
    const double target = u * slots_sum(sh.slots[0], warps);
    const Place at = locate(sh.slots[0], warps, target);
    if (rank == at.g / kRowWarps) {
        const Found f = find_in_slice<DT>(row, warp_slice<DT>(row, at.g, warps), at.base, target, ring, sh.find, kept);
        if (threadIdx.x == 0) a.ids[r] = f.id;
    }
}

}  // namespace qmm

namespace qmm_host {

int row_cluster(long long rows, long long V, int elem_bytes, int ctas, int most) {
    const long long vecs = (V * elem_bytes + 15) / 16, lanes = qmm::kRowThreads;
    int C = 1;
    while (C < 8 && vecs > 2 * C * lanes &&
           (vecs > most * C * lanes || rows * C * 2 <= 148 || (rows * C * 2 <= ctas && vecs > 8 * C * lanes)))
        C *= 2;
    // clusters of 16 find room on fewer SMs: for calls that fit at once
    if (C == 8 && rows * 16 <= 148 && vecs > 16 * lanes) C = 16;
    return C;
}

template <int DT>
static int sample_dt(const qmm::SampleArgs& a, long long rows, cudaStream_t st) {
    const bool filters = a.t_rows || a.k_rows || a.p_rows || a.m_rows || a.t == 0.0 || a.k || a.p < 1.0 || a.m > 0.0;
    if (filters) {
        int C = row_cluster(rows, a.V, qmm::Elem<DT>::kBytes, 8 * 148);
        // a row that may need top-p's bins: no more tokens to a warp than they take
        const bool bins = (a.p_rows || a.p < 1.0) && (a.k_rows || a.k == 0 || a.k > qmm::kRowThreads);
        while (bins && C < 8 && a.V > C * qmm::kRowWarps * (qmm::kBinTokens - 32)) C *= 2;
        return launch_rows(qmm::sample_kernel<DT, true>, qmm::kRowThreads, rows, C, qmm::kSelectSmem, st,
                           "sample launch", a);
    }
    return launch_rows(qmm::sample_kernel<DT, false>, qmm::kRowThreads, rows,
                       row_cluster(rows, a.V, qmm::Elem<DT>::kBytes, 4 * 148), qmm::kDrawSmem, st, "sample launch", a);
}

int launch_sample(const qmm::SampleArgs& a, long long rows, int dtype, cudaStream_t st) {
    if (dtype == QMM_BF16) return sample_dt<0>(a, rows, st);
    if (dtype == QMM_F16) return sample_dt<1>(a, rows, st);
    return sample_dt<2>(a, rows, st);
}

}  // namespace qmm_host
