// logits.cuh -- the core of the operators on rows of logits (sample, top-k,
// speculative acceptance, distillation): how a cluster of CTAs reads a row,
// sums it, orders it and finds a place in it.
//
// A row of V logits belongs to a cluster of C CTAs of 256 threads (C a power
// of two up to 16, by the host's rule).  It is cut into 16-byte vectors at the
// memory's own 16-byte boundaries, so any start of a row (odd V, a view) is
// read with full-width loads; only a first or last vector that holds elements
// of a neighbour is read element by element.  Each warp owns one contiguous
// run of vectors, lanes take every 32nd: the order of warps is the order of
// token ids, so prefix sums over warps are prefix sums over ids.
//
// The order of tokens (logit descending, id ascending) is one 64-bit key: the
// logit's order-preserving bits above the complemented id.  Keys are distinct,
// so every filter is one comparison against a border key.  -0 equals +0; a NaN
// counts as -infinity.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <type_traits>

#include "logits_args.cuh"

namespace qmm {

namespace cg = cooperative_groups;

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kMaxRowWarps = kRowWarps * kMaxCluster;

// QMM_BF16, QMM_F16, QMM_F32
template <int DT>
struct Elem {
    static constexpr int kBytes = DT == 2 ? 4 : 2;
    static constexpr int kVec = 16 / kBytes;
};

// ---- a row in memory ---------------------------------------------------------

template <int DT>
struct Row {
    const char* base;  // the row's start, rounded down to 16 bytes
    int V, shift, nv;  // elements, elements of the first vector before the row, vectors

    QMM_DEVINL Row(const void* logits, long long stride, long long r, int V_) {
        const char* p = static_cast<const char*>(logits) + r * stride * Elem<DT>::kBytes;
        const uintptr_t off = reinterpret_cast<uintptr_t>(p) & 15u;
        base = p - off;
        V = V_;
        shift = (int)(off / Elem<DT>::kBytes);
        nv = (int)(((long long)V + shift + Elem<DT>::kVec - 1) / Elem<DT>::kVec);
    }
    // id of the vector's element 0 (negative, or past V, where the vector sticks out)
    QMM_DEVINL int first(int v) const { return v * Elem<DT>::kVec - shift; }
    QMM_DEVINL bool whole(int v) const { return first(v) >= 0 && first(v) <= V - Elem<DT>::kVec; }
    QMM_DEVINL uint4 load(int v) const;  // elements outside the row read as -infinity
    QMM_DEVINL float at(int i) const;
};

// Logits are read once or twice (the second time from L2): past L1.  Coherent
// loads: the distillation gradient may overwrite its own logits.
QMM_DEVINL uint4 ld_row_v4(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

template <int DT>
QMM_DEVINL uint32_t neg_inf_word() {
    return DT == 0 ? 0xFF80FF80u : DT == 1 ? 0xFC00FC00u : 0xFF800000u;
}

template <int DT>
QMM_DEVINL uint4 Row<DT>::load(int v) const {
    if (whole(v)) return ld_row_v4(base + 16LL * v);
    const int f = first(v);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = neg_inf_word<DT>();
#pragma unroll
    for (int j = 0; j < Elem<DT>::kVec; ++j) {
        const int i = f + j;
        if (i < 0 || i >= V) continue;
        if (DT == 2) {
            w[j & 3] = reinterpret_cast<const volatile uint32_t*>(base)[4LL * v + j];
        } else {
            const uint32_t h = reinterpret_cast<const volatile uint16_t*>(base)[8LL * v + j];
            w[j / 2] = (j & 1) ? (w[j / 2] & 0xFFFFu) | (h << 16) : (w[j / 2] & 0xFFFF0000u) | h;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT>
QMM_DEVINL void store_elem(void* p, long long i, float x) {
    if (DT == 2) static_cast<float*>(p)[i] = x;
    else static_cast<uint16_t*>(p)[i] = Half<DT == 1>::from_f32(x);
}

template <int DT>
QMM_DEVINL float elem_f32(const void* p, long long i) {
    if (DT == 2) return static_cast<const volatile float*>(p)[i];
    return Half<DT == 1>::to_f32(static_cast<const volatile uint16_t*>(p)[i]);
}

template <int DT>
QMM_DEVINL float Row<DT>::at(int i) const {
    return elem_f32<DT>(base, (long long)shift + i);
}

template <int DT>
QMM_DEVINL void decode(const uint4& u, float (&x)[Elem<DT>::kVec]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (DT == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = Half<DT == 1>::lo_f32(w[j]);
            x[2 * j + 1] = Half<DT == 1>::hi_f32(w[j]);
        }
    }
}

// Largest of a vector's elements, NaN ignored (all NaN: NaN in 16 bits, which
// fmaxf then ignores).  Two 16-bit elements to an instruction.
template <int DT>
QMM_DEVINL float vec_max(const uint4& u) {
    if constexpr (DT == 2) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                     fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    } else if constexpr (DT == 0) {
        auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
        const __nv_bfloat162 m = __hmax2(__hmax2(h(u.x), h(u.y)), __hmax2(h(u.z), h(u.w)));
        return fmaxf(__low2float(m), __high2float(m));
    } else {
        auto h = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
        const __half2 m = __hmax2(__hmax2(h(u.x), h(u.y)), __hmax2(h(u.z), h(u.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
}

// ---- keys -----------------------------------------------------------------------

constexpr uint32_t kKeyNegInf = 0x007FFFFFu;  // key32(-infinity); finite logits lie above

QMM_DEVINL uint32_t key32(float x) {
    if (!(x == x)) return kKeyNegInf;
    const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
QMM_DEVINL float key32_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
QMM_DEVINL unsigned long long row_key(float x, int id) {
    return ((unsigned long long)key32(x) << 32) | (0xFFFFFFFFu - (uint32_t)id);
}
QMM_DEVINL int key_id(unsigned long long k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

// ---- weights exp((x - max) / T) ----------------------------------------------------

// In 64 bits.  The largest logit weighs 1 even where it is infinite.
QMM_DEVINL double weight64(float x, float mx, double inv_t) {
    if (x == mx) return 1.0;
    const double w = exp(((double)x - (double)mx) * inv_t);
    return w == w ? w : 0.0;  // NaN logits, and the others beside +infinity
}

QMM_DEVINL float ex2(float a) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}

// log2(e) / T in two floats: the exponent of a fast weight is off by one
// rounding, not by a multiple of the constant's own.
struct Scale {
    float hi, lo;
    QMM_DEVINL explicit Scale(double inv_t) {
        const double c = inv_t * 1.4426950408889634;
        hi = (float)c;
        lo = (float)(c - (double)hi);
    }
    QMM_DEVINL float exponent(float d) const { return fmaf(d, hi, d * lo); }
};

// Differences from the maximum end here: what a masked logit (-infinity, the
// type's lowest value) leaves is a finite exponent and no weight.
constexpr float kFarBelow = -1e30f;
// Temperatures of the fast sums: within them an exponent of kFarBelow is
// finite and weighs nothing.
constexpr double kFastMinT = 1e-6, kFastMaxT = 1e20;
// Bound of the relative error of a fast sum.  A weight: difference and
// exponent rounded once each, |a| ln2 2^-23, where the weighted mean of |a| is
// at most about log2(V) + 2 <= 25: 2.1e-6; ex2.approx 2^-22; up to 8 rescalings
// of a lane's sum, 8 * 2^-22 at worst.  A lane's sum: five roundings within a
// batch of 4 vectors and one per batch, 64 batches at most: 69 * 2^-24 =
// 4.1e-6.  Together 8.4e-6 < 2^-16.
constexpr double kFastEps = 1.0 / 65536.0;
constexpr int kFastVectors = 256;  // vectors to a lane

// Running maximum and sum of weights of one lane.
struct LaneSum {
    float m = -3.402823466e38f, s = 0.0f;  // the lowest finite value: differences from it are no NaN
};

template <int N>
QMM_DEVINL float tree_sum(float (&e)[N]) {
#pragma unroll
    for (int h = N / 2; h >= 1; h /= 2)
#pragma unroll
        for (int j = 0; j < h; ++j) e[j] += e[j + h];
    return e[0];
}

// ---- a cluster's slices --------------------------------------------------------------

struct Slice {
    int begin, end;  // vectors of this warp
    int lane;
};

QMM_DEVINL Slice warp_slice(int nv, int warp, int warps) {
    const int per = (nv + warps - 1) / warps;
    const long long b = (long long)per * warp;
    Slice s;
    s.begin = (int)(b < nv ? b : nv);
    s.end = (int)(b + per < nv ? b + per : nv);
    s.lane = threadIdx.x & 31;
    return s;
}

// f(vector index, vector) over the warp's slice, four loads in flight to a lane.
template <int DT, typename F>
QMM_DEVINL void for_vectors(const Row<DT>& row, const Slice& s, F&& f) {
    int v = s.begin + s.lane;
    for (; v + 96 < s.end; v += 128) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = row.load(v + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) f(v + 32 * i, u[i]);
    }
    for (; v < s.end; v += 32) f(v, row.load(v));
}

// x - m, not below kFarBelow.  A NaN is far below too, or with NAN_THROUGH stays one.
template <bool NAN_THROUGH>
QMM_DEVINL float below(float x, float m) {
    if (!NAN_THROUGH) return fmaxf(x - m, kFarBelow);
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x - m), "f"(kFarBelow));
    return r;
}

// Maximum of the slice's logits in this lane, and with SUM the lane's weights.
// change(vector index, vector) may take elements out (set them to -infinity).
template <int DT, bool SUM, bool NAN_THROUGH, typename F>
QMM_DEVINL float stream_slice(const Row<DT>& row, const Slice& s, const Scale& c, LaneSum& acc, F&& change) {
    constexpr int N = Elem<DT>::kVec;
    float top = -CUDART_INF_F;
    auto batch = [&](const uint4* u, auto n_) {
        constexpr int n = decltype(n_)::value;
        float bm = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < n; ++i) bm = fmaxf(bm, vec_max<DT>(u[i]));
        top = fmaxf(top, bm);
        if (!SUM) return;
        if (bm > acc.m) {
            acc.s *= ex2(c.exponent(below<false>(acc.m, bm)));
            acc.m = bm;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            float e[N];
            decode<DT>(u[i], e);
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] = ex2(c.exponent(below<NAN_THROUGH>(e[j], acc.m)));
            sum += tree_sum<N>(e);
        }
        acc.s += sum;
    };
    int v = s.begin + s.lane;
    for (; v + 96 < s.end; v += 128) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = row.load(v + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) change(v + 32 * i, u[i]);
        batch(u, std::integral_constant<int, 4>());
    }
    for (; v < s.end; v += 32) {
        uint4 u = row.load(v);
        change(v, u);
        batch(&u, std::integral_constant<int, 1>());
    }
    return top;
}

template <int DT, bool SUM>
QMM_DEVINL float stream_slice(const Row<DT>& row, const Slice& s, const Scale& c, LaneSum& acc) {
    return stream_slice<DT, SUM, false>(row, s, c, acc, [](int, uint4&) {});
}

// ---- exchange between the warps of a cluster ---------------------------------------------

QMM_DEVINL float warp_max(float x) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
template <typename T>
QMM_DEVINL T warp_sum(T x) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

// Every warp's value to every CTA of the cluster: slot g of `slots` (the same
// shared array in each CTA) is warp g's.  The caller syncs the cluster before
// it reads, and alternates between two arrays from one exchange to the next.
template <typename T>
QMM_DEVINL void all_gather(cg::cluster_group& cl, T* slots, int g, const T& value) {
    const int lane = threadIdx.x & 31;
    if (lane < (int)cl.num_blocks()) *cl.map_shared_rank(slots + g, lane) = value;
}

// Sum of n slots in their order, the same in every thread.
QMM_DEVINL double slots_sum(const double* slots, int n) {
    const int lane = threadIdx.x & 31;
    double x = 0.0;
    for (int i = lane; i < n; i += 32) x += slots[i];
    return warp_sum(x);
}

struct Place {
    int g;        // slot
    double base;  // sum of the slots before it
};

QMM_DEVINL float slots_max(const float* slots, int n) {
    float x = -CUDART_INF_F;
    for (int i = threadIdx.x & 31; i < n; i += 32) x = fmaxf(x, slots[i]);
    return warp_max(x);
}

// A warp's sum of weights against the row's maximum mx.
QMM_DEVINL double warp_mass(const LaneSum& acc, const Scale& c, float mx) {
    return warp_sum((double)acc.s * (double)ex2(c.exponent(below<false>(acc.m, mx))));
}

// The first slot at which the running sum passes `target`, or the last slot
// that holds anything.  Called by whole warps; equal in every warp.
QMM_DEVINL Place locate(const double* slots, int n, double target) {
    const int lane = threadIdx.x & 31;
    const int per = (n + 31) / 32;  // 1 .. 4 consecutive slots to a lane
    double x[kMaxRowWarps / 32], run = 0.0;
#pragma unroll
    for (int i = 0; i < kMaxRowWarps / 32; ++i) {
        const int at = lane * per + i;
        x[i] = i < per && at < n ? slots[at] : 0.0;
        run += x[i];
    }
    double incl = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += y;
    }
    double base = __shfl_up_sync(~0u, incl, 1);
    if (lane == 0) base = 0.0;
    int hit = -1, last = -1;
    double hit_base = 0.0, last_base = 0.0;
#pragma unroll
    for (int i = 0; i < kMaxRowWarps / 32; ++i) {
        if (x[i] > 0.0) {
            last = lane * per + i;
            last_base = base;
            if (hit < 0 && base + x[i] > target) {
                hit = lane * per + i;
                hit_base = base;
            }
        }
        base += x[i];
    }
    const unsigned hits = __ballot_sync(~0u, hit >= 0), lasts = __ballot_sync(~0u, last >= 0);
    Place p;
    if (hits) {
        p.g = __shfl_sync(~0u, hit, __ffs(hits) - 1);
        p.base = __shfl_sync(~0u, hit_base, __ffs(hits) - 1);
    } else if (lasts) {
        p.g = __shfl_sync(~0u, last, 31 - __clz(lasts));
        p.base = __shfl_sync(~0u, last_base, 31 - __clz(lasts));
    } else {
        p.g = -1;
        p.base = 0.0;
    }
    return p;
}

// Within one warp's slice: the first id at which base + the running sum of
// weights passes `target`, with the sums just before and after it; the last id
// of any weight if none does.  weight(id, logit) is in 64 bits.
struct Found {
    int id;
    double before, after;
};

template <int DT, typename W>
QMM_DEVINL Found find_in_slice(const Row<DT>& row, const Slice& s, double base, double target, W&& weight) {
    constexpr int N = Elem<DT>::kVec;
    Found found{-1, 0.0, 0.0};
    uint4 next = make_uint4(0, 0, 0, 0);
    if (s.begin + s.lane < s.end) next = row.load(s.begin + s.lane);
    for (int v0 = s.begin; v0 < s.end; v0 += 32) {
        const int v = v0 + s.lane;
        const uint4 cur = next;
        if (v + 32 < s.end) next = row.load(v + 32);
        double w[N], mine = 0.0;
        float x[N];
        decode<DT>(cur, x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int id = row.first(v) + j;
            w[j] = v < s.end && id >= 0 && id < row.V ? weight(id, x[j]) : 0.0;
            mine += w[j];
        }
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(~0u, incl, o);
            if (s.lane >= o) incl += y;
        }
        const unsigned hits = __ballot_sync(~0u, mine > 0.0 && base + incl > target);
        const unsigned any = __ballot_sync(~0u, mine > 0.0);
        if (any) {
            // the first lane that passes, else the last with a weight (kept for the end)
            const int src = hits ? __ffs(hits) - 1 : 31 - __clz(any);
            double run = base + incl - mine;
            Found f{-1, 0.0, 0.0};
            bool done = false;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (w[j] > 0.0 && !done) {
                    f.id = row.first(v) + j;
                    f.before = run;
                    f.after = run + w[j];
                    run += w[j];
                    done = run > target;
                }
            }
            found.id = __shfl_sync(~0u, f.id, src);
            found.before = __shfl_sync(~0u, f.before, src);
            found.after = __shfl_sync(~0u, f.after, src);
            if (hits) return found;
        }
        base += __shfl_sync(~0u, incl, 31);
    }
    return found;
}

}  // namespace qmm

namespace qmm_host {

// CTAs to a row: enough that a lane holds few vectors, and that a call of few
// rows reaches every SM.
int row_cluster(long long rows, long long V, int elem_bytes);

// Launch `kernel` over rows * C CTAs of kRowThreads in clusters of C.
template <typename... P, typename... A>
int launch_rows(void (*kernel)(P...), long long rows, int C, size_t smem, cudaStream_t st, const char* what,
                A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * C));
    cfg.blockDim = dim3(qmm::kRowThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)C;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cudaError_t e = cudaSuccess;
    if (C > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return cuda_status(e, what);
}

}  // namespace qmm_host
