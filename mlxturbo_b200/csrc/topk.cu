// topk.cu -- the k largest logits of a row with their ids, and the row's
// log-sum-exp (ops.topk): what a distillation takes from its teacher and a
// sharded lm_head exchanges instead of its logits.
//
// One pass over memory.  The k-th largest of maxima of groups of lanes (twice k
// of them or more) bounds the k-th largest logit from below, and about 1.4 k
// logits reach it.  A lane has kept where its two largest vectors are, reads
// them again (from L2), and CTA 0 sorts what is found.  Rows where too many
// reach the bound (many equal logits, k near the number of threads) search the
// border key and collect above it.
//
// Bound by memory and, with the log-sum-exp, by the exponential unit (eight of
// them to 16 bytes: 111 of 245 us); what keeps it from its floor is the tail of
// a row, 10 us in which its CTAs read nothing.  B200, V 248320: 2011 rows, k 64,
// with log-sum-exp 245 us (floor 153); 5 rows, k 20, 10 us.

#include "logits_select.cuh"

namespace qmm {

template <int DT, bool LSE>
__global__ void __launch_bounds__(kRowThreads, 4) topk_kernel(const TopkArgs a) {
    extern __shared__ uint4 memory[];
    SelectShared& sh = *reinterpret_cast<SelectShared*>(memory + kRing * kRowThreads);
    const Ring ring = reinterpret_cast<Ring>(memory);
    cg::cluster_group cl = cg::this_cluster();
    cl.barrier_arrive();  // waited for before the first access to another CTA
    if (threadIdx.x == 0) sh.n_cand = 0;
    if (LSE) fill_table(sh.table);
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), warps = C * kRowWarps;
    const int g = rank * kRowWarps + (threadIdx.x >> 5);
    const long long r = blockIdx.x / C;
    const Row<DT> row(a.logits, a.stride, r, a.V);
    const Slice s = warp_slice<DT>(row, g, warps);
    const Scale c(a.inv_t);

    LaneSum acc;
    const LaneTop top = stream_slice<DT, LSE, true>(row, s, c, acc);
    const bool listed = a.k <= C * kRowThreads;
    const int lanes = lanes_to_group(warps, a.k);
    const WarpStat stat = warp_stat(top.first, acc, LSE);
    cl.barrier_wait();
    if (LSE) all_gather(cl, sh.stats, g, stat);
    if (listed) publish_maxima(cl, sh, g, lanes, top.first);
    cl.sync();
    float mx = 0.0f;
    double total = 0.0;
    if (LSE) row_stat(sh.stats, warps, c, mx, total, nullptr);
    const uint32_t bound = listed ? kth_bound(sh, warps * (32 / lanes), a.k) : 0;
    const Weight64 weight(sh.table, mx, 1.0 / a.inv_t, a.inv_t);
    if (LSE && fabsf(mx) != CUDART_INF_F && !(c.fast(mx, 1.0 / a.inv_t) && total >= 0.5 && total < CUDART_INF)) {
        double mass = 0.0;  // a NaN among the logits, or none above a mask's lowest value
        for_vectors_slow<DT>(row, s, ring, [&](int, const uint4& q) {
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
    }
    if (LSE && rank == 0 && threadIdx.x < 32) {
        // no finite maximum: the sum is that of the largest alone
        const double l = mx == -CUDART_INF_F || mx == CUDART_INF_F ? (double)mx : (double)mx * a.inv_t + log(total);
        if (threadIdx.x == 0) a.lse[r] = (float)l;
    }
    uint32_t n = kCand + 1;
    if (listed) {
        const uint32_t mine = push_candidates<DT>(cl, sh, row, s, top, bound);
        all_gather(cl, sh.found, g, mine);
        cl.sync();
        n = 0;
        for (int i = s.lane; i < warps; i += 32) n += sh.found[i];
        n = warp_sum(n);
    }
    if (n > kCand) {  // the border, then the k tokens from it on
        // the search takes logits up to its maximum: infinite ones too
        const unsigned long long border = border_key<DT, false>(cl, sh, row, s, g, warps, ring,
                                                                Weight64(sh.table, CUDART_INF_F, 1.0, 1.0),
                                                                (unsigned long long)kKeyNegInf << 32, (double)a.k);
        cl.sync();
        if (threadIdx.x == 0) sh.n_cand = 0;
        cl.sync();
        append_slice<DT>(cl, sh, row, s, 0, 0xFFFFFFFFu, border);
        cl.sync();
        n = (uint32_t)a.k;
    }
    if (rank != 0) return;
    sort_candidates(sh.cand, (int)n);
    for (int i = threadIdx.x; i < a.k; i += kRowThreads) {
        const int id = key_id(sh.cand[i]);
        float x = key32_value((uint32_t)(sh.cand[i] >> 32));
        if (x == 0.0f) x = row.at(id);  // -0 has the key of +0
        store_elem<DT>(a.values, r * a.k + i, x);
        a.ids[r * a.k + i] = id;
    }
}

}  // namespace qmm

namespace qmm_host {

template <int DT>
static int topk_dt(const qmm::TopkArgs& a, long long rows, cudaStream_t st) {
    // One CTA holds a long row's maxima as well as two (2011 rows of 248320, k 64: 248 us against 274), if they
    // are twice k.
    int C = row_cluster(rows, a.V, qmm::Elem<DT>::kBytes, 4 * 148, 128);
    while (C < 8 && C * qmm::kRowThreads < 2 * a.k && (long long)a.V * qmm::Elem<DT>::kBytes > 32LL * C * qmm::kRowThreads)
        C *= 2;
    if (a.lse) return launch_rows(qmm::topk_kernel<DT, true>, qmm::kRowThreads, rows, C, qmm::kSelectSmem, st, "topk launch", a);
    return launch_rows(qmm::topk_kernel<DT, false>, qmm::kRowThreads, rows, C, qmm::kSelectSmem, st, "topk launch", a);
}

int launch_topk(const qmm::TopkArgs& a, long long rows, int dtype, cudaStream_t st) {
    if (dtype == QMM_BF16) return topk_dt<0>(a, rows, st);
    if (dtype == QMM_F16) return topk_dt<1>(a, rows, st);
    return topk_dt<2>(a, rows, st);
}

}  // namespace qmm_host
