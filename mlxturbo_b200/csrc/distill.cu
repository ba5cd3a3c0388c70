// distill.cu -- Kullback-Leibler divergence of a row of logits from a
// teacher's top logits, and its gradient (ops.distill_loss).
//
// The teacher's list of a row is k (logit, id) pairs; ids outside [0, V) are
// empty places.  p are the listed probabilities: exp(t_j / tau) over their
// sum, or, with the teacher's log-sum-exp given, over the whole sum, the rest
// 1 - sum p being one more class that holds every token not listed.  With
// q = softmax(l / tau), Z its sum and O the part of it that is not listed:
//
//   loss  = sum_j p_j (log p_j - log q_j)  [ + rest (log rest - log (O / Z)) ]
//   dloss/dl_i = (q_i - p_i) / tau                     listed tokens
//              = e_i (1 / Z  [ - rest / O ]) / tau     the others, e_i / Z = q_i
//
// j counts distinct ids: p_j is the sum over the entries that name the id.
//
// O is summed on its own (a bit to an element marks the listed ones), not as a
// difference: it may be a billionth of Z.  Its weights are taken against the
// largest logit that is not listed, so neither O nor rest / O leaves the range
// of 32 bits.  The loss, too, is made of differences to the largest listed
// logit: of logits near a type's limit 64 bits would keep no digit.  A gradient
// below 2^-126 times its row's weight / tau may come out as 0: the exponentials
// have no smaller values.
//
// Bound by memory: the loss reads the logits once, the gradient reads and
// writes them once.  Loss and gradient in one call are one launch, a cluster to
// a row, which reads the row twice; of the second reading L2 has a third, since
// the rows at work (296 of 497 KB) are more than it holds, and fewer rows at
// work, by more CTAs to a row, cost more in their steps than they save (2048 rows
// of 248320 by 2, 4, 8 CTAs: 464, 500, 767 us of the device's time).  B200,
// V 248320, bf16: loss of 333 rows 43 to 45 us (floor 25), of 1024 96 us (78);
// backward of 1024 rows 161 us, 96% of the copy rate; both of 2048 rows in one
// launch 485 to 490 us through the public call (floor 311 with one reading, 466
// with two).

#include "logits.cuh"

namespace qmm {

// Temperatures below the largest logit at which a token has no weight, whatever
// their number: exp(-700) is 1e-304.
constexpr double kNoWeight = -700.0;

// A CTA: eight warps read logits, a ninth works through the list meanwhile.
constexpr int kDistillThreads = kRowThreads + 32;

struct DistillShared {
    WarpStat stats[kMaxRowWarps];
    double mass;   // sum p
    double cross;  // sum p (log p - (l - base) / tau), for the loss
    double part;   // sum over distinct listed tokens of exp((l - best) / tau)
    float best;    // largest listed logit

    // what the loss' logits are counted from
    QMM_DEVINL static double base(float best) { return fabsf(best) < CUDART_INF_F ? (double)best : 0.0; }
    int twice;     // an id is listed more than once
};

// The list, in dynamic shared memory.
struct List {
    double* logp;
    float* x;   // the student's logits
    int* id;    // or -1
    int* slot;  // place in the table of distinct ids
    int *table, *owner;
    int size;  // of the table

    static __host__ __device__ int table_size(int k) {
        int n = 2;
        while (n < 2 * k) n <<= 1;
        return n;
    }
    static __host__ __device__ size_t bytes(int k) { return (size_t)k * 20 + (size_t)table_size(k) * 8; }
    QMM_DEVINL List(void* memory, int k)
        : logp(static_cast<double*>(memory)), x(reinterpret_cast<float*>(logp + k)), id(reinterpret_cast<int*>(x + k)),
          slot(id + k), table(slot + k), owner(table + table_size(k)), size(table_size(k)) {}
};

// The ids of the list, by one warp; four loads of a lane at a time, as below.
QMM_DEVINL void list_ids(const DistillArgs& a, const List& li, long long r) {
    for (int j0 = threadIdx.x & 31; j0 < a.k; j0 += 128) {
        long long id[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long at = r * a.k + min(j0 + 32 * i, a.k - 1);
            id[i] = a.ti_bytes == 8 ? __ldg(static_cast<const long long*>(a.ti) + at)
                                    : (long long)__ldg(static_cast<const int*>(a.ti) + at);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j0 + 32 * i < a.k) li.id[j0 + 32 * i] = id[i] >= 0 && id[i] < a.V ? (int)id[i] : -1;
    }
    __syncwarp();
}

// The rest of it, by one warp: log p and the student's logits; entries of one
// id share a slot whose owner is the first of them; the sums (LOSS: the loss' too).
template <int DT, bool TAIL, bool LOSS>
QMM_DEVINL void list_sums(const DistillArgs& a, DistillShared& sh, const List& li, const Row<DT>& row, long long r) {
    const int lane = threadIdx.x & 31;
    double top = -CUDART_INF;
    float best = -CUDART_INF_F;
    for (int j0 = lane; j0 < a.k; j0 += 128) {
        float t[4], x[4];
        int id[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = min(j0 + 32 * i, a.k - 1);
            const long long at = r * a.k + j;
            id[i] = li.id[j];
            t[i] = a.tv_dtype == 2 ? __ldg(static_cast<const float*>(a.tv) + at)
                   : a.tv_dtype == 1 ? Half<true>::to_f32(__ldg(static_cast<const uint16_t*>(a.tv) + at))
                                     : Half<false>::to_f32(__ldg(static_cast<const uint16_t*>(a.tv) + at));
            x[i] = id[i] >= 0 ? row.at(id[i]) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (j0 + 32 * i >= a.k) break;
            const double l = id[i] >= 0 ? (double)t[i] * a.inv_t : -CUDART_INF;
            li.x[j0 + 32 * i] = x[i];
            li.logp[j0 + 32 * i] = l;
            top = fmax(top, l);  // a NaN shows in the sums
            if (id[i] >= 0) best = fmaxf(best, x[i]);
        }
    }
    for (int i = lane; i < li.size; i += 32) {
        li.table[i] = -1;
        li.owner[i] = kMaxList;
    }
    __syncwarp();
    bool twice = false;
    for (int j = lane; j < a.k; j += 32) {
        const int id = li.id[j];
        if (id < 0) continue;
        int h = (int)((uint32_t)id * 2654435761u >> 16) & (li.size - 1);
        for (;;) {
            const int was = atomicCAS(&li.table[h], -1, id);
            twice |= was == id;
            if (was == -1 || was == id) break;
            h = (h + 1) & (li.size - 1);
        }
        li.slot[j] = h;
        atomicMin(&li.owner[h], j);
    }
    __syncwarp();
    twice = __any_sync(~0u, twice);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmax(top, __shfl_xor_sync(~0u, top, o));
    best = warp_max(best);
    double norm = 0.0;
    if (TAIL) {
        norm = (double)a.tlse[r];
    } else if (top != -CUDART_INF) {  // else nothing is listed
        double sum = 0.0;
        for (int j = lane; j < a.k; j += 32) sum += exp(li.logp[j] - top);
        norm = top + log(warp_sum(sum));
    }
    const double base = DistillShared::base(best);
    double mass = 0.0, cross = 0.0, part = 0.0;
    for (int j = lane; j < a.k; j += 32) {
        const double lp = li.logp[j] - norm, p = exp(lp);
        li.logp[j] = lp;
        mass += p;
        if (li.id[j] < 0) continue;
        if (LOSS && !twice && p != 0.0) cross += p * (lp - ((double)li.x[j] - base) * a.inv_t);
        // (where the list holds nothing but masked tokens, best is -infinity as they are)
        if (TAIL && li.owner[li.slot[j]] == j && li.x[j] != -CUDART_INF_F)
            part += exp(((double)li.x[j] - (double)best) * a.inv_t);
    }
    if (LOSS && twice) {  // an id's entries added up before the logarithm
        __syncwarp();
        for (int j = lane; j < a.k; j += 32) {
            const int id = li.id[j];
            if (id < 0 || li.owner[li.slot[j]] != j) continue;
            double p = exp(li.logp[j]);
            for (int i = j + 1; i < a.k; ++i)
                if (li.id[i] == id) p += exp(li.logp[i]);
            if (p != 0.0) cross += p * (log(p) - ((double)li.x[j] - base) * a.inv_t);
        }
    }
    mass = warp_sum(mass);
    cross = warp_sum(cross);
    if (TAIL) part = warp_sum(part);
    if (lane == 0) {
        sh.mass = mass;
        sh.cross = cross;
        sh.part = part;
        sh.best = best;
        sh.twice = twice;
    }
}

// Every listed element of this vector set to -infinity; bit j of m is element j.
template <int DT>
QMM_DEVINL void take_out(uint4& u, uint32_t m) {
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == 2) {
            if (m >> i & 1) w[i] = 0xFF800000u;
        } else {
            if (m >> (2 * i) & 1) w[i] = (w[i] & 0xFFFF0000u) | (neg_inf_word<DT>() & 0xFFFFu);
            if (m >> (2 * i + 1) & 1) w[i] = (w[i] & 0xFFFFu) | (neg_inf_word<DT>() & 0xFFFF0000u);
        }
    }
    u = make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT>
QMM_DEVINL uint4 encode(const float (&x)[Elem<DT>::kVec]) {
    if constexpr (DT == 2) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else {
        using H = Half<DT == 1>;
        return make_uint4(H::pack2(x[0], x[1]), H::pack2(x[2], x[3]), H::pack2(x[4], x[5]), H::pack2(x[6], x[7]));
    }
}

// A finite reference that the fast weights do not take, its E's rounding being
// above a half: rows masked throughout with a type's lowest value.
QMM_DEVINL bool out_of_range(float ref, const Scale& c) {
    return fabsf(ref * c.c) > 16777216.0f && fabsf(ref) < CUDART_INF_F;
}

// TAIL: the teacher's log-sum-exp is given.  MODE kBackward needs no cluster.
template <int DT, bool TAIL, int MODE>
__global__ void __launch_bounds__(kDistillThreads, MODE == kBackward ? 3 : 4)
    distill_kernel(const DistillArgs a, int C) {
    __shared__ DistillShared sh;
    extern __shared__ uint4 memory[];
    const StreamRing ring = reinterpret_cast<StreamRing>(memory);  // of the passes that write
    const List li(memory + (MODE == kLoss ? 0 : kStream * kRowThreads), a.k);
    // TAIL: a byte to a vector of this CTA
    uint32_t* const marks = reinterpret_cast<uint32_t*>(li.owner + li.size);
    constexpr int N = Elem<DT>::kVec;
    cg::cluster_group cl = cg::this_cluster();
    if (MODE != kBackward) cl.barrier_arrive();
    const int rank = (int)(blockIdx.x % C), warps = C * kRowWarps, warp = threadIdx.x >> 5;
    const bool reader = warp < kRowWarps;
    const int g = rank * kRowWarps + warp;
    const long long r = blockIdx.x / C;
    const Row<DT> row(a.logits, a.stride, r, a.V);
    const int per = (row.nv + warps - 1) / warps, cta_begin = per * kRowWarps * rank;
    const int cta_end = cta_begin + per * kRowWarps;
    const Slice s = warp_slice<DT>(row, g, warps);
    const Scale c(a.inv_t);
    const float tlse = TAIL ? a.tlse[r] : 0.0f;
    // a teacher's row that is masked throughout carries no loss
    const bool none = TAIL && tlse == -CUDART_INF_F;
    const float weight = none ? 0.0f : a.weight ? a.weight[r] : 1.0f;

    float ref, mx;       // the others' reference; the row's maximum
    double others, sum;  // factor of the others' gradient; sum against mx
    if (MODE == kBackward) {
        const float4 st = a.stats[r];
        ref = st.x;
        others = st.y;
        mx = st.z;
        sum = st.w;
        if (!reader && weight != 0.0f) {
            list_ids(a, li, r);
            list_sums<DT, TAIL, false>(a, sh, li, row, r);
        }
    } else {
        if (!reader) list_ids(a, li, r);
        if (TAIL) {
            for (int i = threadIdx.x; i < (per * kRowWarps + 3) / 4; i += kDistillThreads) marks[i] = 0;
            __syncthreads();
            if (!reader) {
                for (int j = s.lane; j < a.k; j += 32) {
                    const int at = li.id[j] + row.shift, v = at / N - cta_begin;
                    if (li.id[j] >= 0 && v >= 0 && v < per * kRowWarps)
                        atomicOr(&marks[v / 4], 1u << (8 * (v & 3) + at % N));
                }
            }
            __syncthreads();
        }
        const uint8_t* mark = reinterpret_cast<const uint8_t*>(marks);
        WarpStat stat{};
        if (reader) {
            LaneSum acc;
            auto unlisted = [&](int v, uint4& u) {
                if (TAIL) {
                    const uint32_t m = mark[v - cta_begin];
                    if (m) take_out<DT>(u, m);
                }
            };
            LaneTop top;
            if constexpr (MODE == kLoss) top = stream_slice<DT, true, false>(row, s, c, acc, unlisted);
            else top = stream_slice<DT, true, false>(row, s, c, acc, unlisted, ring);
            stat = warp_stat(top.first, acc);
        } else {
            list_sums<DT, TAIL, true>(a, sh, li, row, r);
        }
        cl.barrier_wait();
        if (reader) all_gather(cl, sh.stats, g, stat);
        cl.sync();
        double s_ref;
        row_stat(sh.stats, warps, c, ref, s_ref, nullptr);
        if (ref == -CUDART_INF_F) s_ref = 0.0;
        if (out_of_range(ref, c)) {
            double share = 0.0;
            if (reader) {
                for_vectors_rare<DT>(row, s, [&](int v, uint4 u) {
                    if (TAIL && mark[v - cta_begin]) take_out<DT>(u, mark[v - cta_begin]);
                    float x[N];
                    decode<DT>(u, x);
#pragma unroll
                    for (int j = 0; j < N; ++j) share += exp(((double)x[j] - (double)ref) * a.inv_t);
                });
            }
            share = warp_sum(share);
            cl.sync();
            if (reader) all_gather(cl, sh.stats, g, WarpStat{share, 0.0f, 0.0f});
            cl.sync();
            s_ref = 0.0;
            for (int i = s.lane; i < warps; i += 32) s_ref += sh.stats[i].s;
            s_ref = warp_sum(s_ref);
        }
        if (MODE == kLoss && (rank != 0 || reader)) return;
        // the list's part of the sum
        const double mass = sh.mass;
        double rest = 0.0;
        mx = ref;
        sum = s_ref;
        if (TAIL) {
            mx = fmaxf(ref, sh.best);
            // one of the two is 1; the other to some digits of 32 bits
            const float lift = ref == -CUDART_INF_F ? 0.0f : expf((float)(((double)ref - (double)mx) * a.inv_t));
            const float down = sh.best == -CUDART_INF_F ? 0.0f : expf((float)(((double)sh.best - (double)mx) * a.inv_t));
            sum = s_ref * (double)lift + sh.part * (double)down;
            rest = mass < 1.0 ? 1.0 - mass : mass >= 1.0 ? 0.0 : mass;
            // A list of all that is not masked leaves a rest of rounding alone: of the log-sum-exp's 32 bits and of
            // the fast sums it may come from.
            if (((double)ref - (double)mx) * a.inv_t < kNoWeight &&
                rest <= 2.0 * kFastEps + fabs((double)tlse) * (1.0 / 8388608.0))
                rest = 0.0;
            others = (double)lift / sum - (s_ref > 0.0 ? rest / s_ref : 0.0);
            if (ref == -CUDART_INF_F) others = 0.0;  // no token that is not listed has any probability
        } else {
            others = mass == 0.0 ? 0.0 : 1.0 / sum;
        }
        if (rank == 0 && threadIdx.x == kRowThreads) {
            double loss = sh.cross;
            if (mass != 0.0) loss += mass * (((double)mx - DistillShared::base(sh.best)) * a.inv_t + log(sum));
            if (TAIL && rest != 0.0) {
                const double log_other = ref == -CUDART_INF_F
                                             ? -CUDART_INF
                                             : ((double)ref - (double)mx) * a.inv_t + log(s_ref) - log(sum);
                loss += rest * (log(rest) - log_other);
            }
            a.loss[r] = none ? 0.0f : (float)loss;
            if (MODE == kLoss && a.stats) a.stats[r] = make_float4(ref, (float)others, mx, (float)sum);
        }
        if (MODE == kLoss) return;
    }

    // gradient
    char* const out = static_cast<char*>(a.grad) + r * a.grad_stride * Elem<DT>::kBytes;
    const bool aligned = ((reinterpret_cast<uintptr_t>(out) - row.shift * Elem<DT>::kBytes) & 15u) == 0;
    auto store = [&](int v, const float (&y)[N]) {
        const int f = row.first(v);
        if (aligned && row.whole(v)) {
            __stcs(reinterpret_cast<uint4*>(out + (long long)f * Elem<DT>::kBytes), encode<DT>(y));
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (f + j >= 0 && f + j < row.V) store_elem<DT>(out, f + j, y[j]);
        }
    };
    const double scale = (double)weight * a.inv_t;
    const float factor = weight == 0.0f ? 0.0f : (float)(scale * others);
    if (reader) {
        if (factor == 0.0f) {  // a row that carries no loss, or one whose other tokens get none: whatever their logits
            const float zero[N] = {};
            for (int v = s.begin + s.lane; v < s.end; v += 32) store(v, zero);
            if (s.lane == 0 && s.head >= 0) store(s.head, zero);
            if (s.lane == 0 && s.tail >= 0) store(s.tail, zero);
        } else if (out_of_range(ref, c)) {
            for_vectors_rare<DT>(row, s, [&](int v, const uint4& u) {
                float x[N];
                decode<DT>(u, x);
#pragma unroll
                for (int j = 0; j < N; ++j)
                    x[j] = (float)(scale * others * exp(((double)x[j] - (double)ref) * a.inv_t));
                store(v, x);
            });
        } else {
            const float e = ceilf(ref * c.c), scaled = (float)(scale * others * c.against(e, ref));
            for_vectors<DT>(row, s, [&](int v, const uint4& u) {
                float x[N];
                decode<DT>(u, x);
#pragma unroll
                for (int j = 0; j < N; ++j) x[j] = scaled * ex2(fmaf(x[j], c.c, -e));
                store(v, x);
            }, ring);
        }
    }
    if (weight == 0.0f) return;
    __syncthreads();  // the listed tokens' values after the others' formula has been written in their place
    const bool empty = !TAIL && sh.mass == 0.0;
    for (int j = threadIdx.x; j < a.k; j += kDistillThreads) {
        const int id = li.id[j];
        if (id < 0 || li.owner[li.slot[j]] != j) continue;
        const int v = (id + row.shift) / N;
        if (v < cta_begin || v >= cta_end) continue;
        double p = exp(li.logp[j]);
        if (sh.twice) {
            for (int i = j + 1; i < a.k; ++i)
                if (li.id[i] == id) p += exp(li.logp[i]);
        }
        const double q = empty ? 0.0 : exp(((double)li.x[j] - (double)mx) * a.inv_t) / sum;
        store_elem<DT>(out, id, (float)(scale * (q - p)));
    }
}

}  // namespace qmm

namespace qmm_host {

template <int DT, bool TAIL, int MODE>
static int distill_launch(const qmm::DistillArgs& a, long long rows, cudaStream_t st) {
    const int C = row_cluster(rows, a.V, qmm::Elem<DT>::kBytes, (MODE == qmm::kBackward ? 3 : 4) * 148,
                              MODE == qmm::kLoss ? 128 : 64);
    size_t smem = qmm::List::bytes(a.k);
    if (MODE != qmm::kLoss) smem += qmm::kStream * qmm::kRowThreads * sizeof(uint4);
    if (MODE == qmm::kBackward)  // CTAs on their own
        return launch_rows(qmm::distill_kernel<DT, TAIL, MODE>, qmm::kDistillThreads, rows * C, 1, smem, st,
                           "distill launch", a, C);
    if (TAIL) {
        const long long vecs = (a.V + 2LL * qmm::Elem<DT>::kVec - 2) / qmm::Elem<DT>::kVec;  // any start of a row
        const int warps = C * qmm::kRowWarps;
        smem += (size_t)(((vecs + warps - 1) / warps) * qmm::kRowWarps + 3) / 4 * 4;
        if (smem > 200 * 1024) {
            set_error("distill: V=%d is too long for teacher_logsumexp", a.V);
            return QMM_EUNSUPPORTED;
        }
    }
    return launch_rows(qmm::distill_kernel<DT, TAIL, MODE>, qmm::kDistillThreads, rows, C, smem, st, "distill launch", a,
                       C);
}

template <int DT, bool TAIL>
static int distill_mode(const qmm::DistillArgs& a, long long rows, int mode, cudaStream_t st) {
    if (mode == qmm::kLoss) return distill_launch<DT, TAIL, qmm::kLoss>(a, rows, st);
    if (mode == qmm::kLossGrad) return distill_launch<DT, TAIL, qmm::kLossGrad>(a, rows, st);
    return distill_launch<DT, TAIL, qmm::kBackward>(a, rows, st);
}

template <int DT>
static int distill_dt(const qmm::DistillArgs& a, long long rows, int mode, cudaStream_t st) {
    return a.tlse ? distill_mode<DT, true>(a, rows, mode, st) : distill_mode<DT, false>(a, rows, mode, st);
}

int launch_distill(const qmm::DistillArgs& a, long long rows, int dtype, int mode, cudaStream_t st) {
    if (dtype == QMM_BF16) return distill_dt<0>(a, rows, mode, st);
    if (dtype == QMM_F16) return distill_dt<1>(a, rows, mode, st);
    return distill_dt<2>(a, rows, mode, st);
}

}  // namespace qmm_host
