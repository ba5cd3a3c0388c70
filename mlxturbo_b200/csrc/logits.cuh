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
    QMM_DEVINL uint4 load_whole(int v) const;
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
QMM_DEVINL uint4 Row<DT>::load_whole(int v) const {
    return ld_row_v4(base + 16LL * v);
}

template <int DT>
QMM_DEVINL uint4 Row<DT>::load(int v) const {
    if (whole(v)) return load_whole(v);
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

QMM_DEVINL float ex2(float a) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}

// In 64 bits: 2^t, t = (x - max) log2(e) / T, as a table's 2^(j/32) times the
// Taylor polynomial of 2^r, |r| <= 1/64 (the term left out is below 3e-15),
// with the whole part added to the exponent: 10 operations of the 64-bit pipe
// and no branch, so the elements of a vector overlap (with exp() and its
// branches a vector of 8 took 3.4 us of a warp's time).  That pipe takes a cycle
// of an SM to 32 elements, so a pass over a row costs four times what reading
// 16-bit logits does; summing all rows of a call this way took 200 us for 512
// rows of 248320, against 180 with fast sums and 64 bits for the open rows only.
// The largest logit weighs 1 even where it is infinite; below 2^-1000, and for
// NaN, there is no weight.
struct Weight64 {
    const double* table;  // 2^(j/32), j = 0 .. 31, in shared memory
    double c, b, inv_t;
    float mx, least;

    // inv_t = 1 / T
    QMM_DEVINL Weight64(const double* table_, float mx_, double T, double inv_t_)
        : table(table_), c(inv_t_ * 1.4426950408889634), b(-(double)mx_ * c), inv_t(inv_t_), mx(mx_),
          least(mx_ - 693.0f * (float)T) {}  // 1000 ln2

    QMM_DEVINL double operator()(float x) const {
        const double t = fma((double)x, c, b);
        const double magic = 6755399441055744.0 / 32.0;  // 1.5 * 2^52 / 32: sums are whole 32nds
        const double k = t + magic;
        const double r = t - (k - magic);
        const int n = __double2loint(k);
        // ln2^i / i!
        double p = fma(r, 1.3333558146428443e-3, 9.618129107628477e-3);
        p = fma(r, p, 5.550410866482158e-2);
        p = fma(r, p, 2.4022650695910072e-1);
        p = fma(r, p, 6.931471805599453e-1);
        p = fma(r, p, 1.0) * table[n & 31];
        const double w = __hiloint2double(__double2hiint(p) + ((n >> 5) << 20), __double2loint(p));
        return x == mx ? 1.0 : x > least ? w : 0.0;
    }
};

QMM_DEVINL void fill_table(double* table) {
    if (threadIdx.x < 32) table[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
}

// Fast weights: 2^(x c - E) with c = log2(e) / T in 32 bits and a whole number
// E, so one multiply-add, and every change of reference is exact.
// Bound of the relative error of a fast sum: the exponent's rounding and c's
// own, |a| ln2 (2^-24 + 2^-24) with a weighted mean of |a| of at most about
// log2(V) + 2 <= 30: 2.5e-6; ex2.approx 2^-22; five roundings within a batch of
// 4 vectors, 3.0e-7; batches are added in 64 bits.  Together 3.1e-6 < 2^-18.
constexpr double kFastEps = 1.0 / 262144.0;
// It stands for finite maxima up to kFastMax and these temperatures.  Beyond, or
// where a NaN or an infinity enters, a sum comes out as NaN or outside
// [0.5, inf) and is made in 64 bits; so it does where E is so large (2^31 and
// more) that its own rounding leaves the exponent's range.
constexpr float kFastMax = 1e29f;
constexpr double kFastMinT = 1e-6, kFastMaxT = 1e6;

struct Scale {
    float c;
    QMM_DEVINL explicit Scale(double inv_t) : c((float)(inv_t * 1.4426950408889634)) {}
    // what turns a sum against E = ceil(mx c) into one against the weight of mx
    QMM_DEVINL double against(float e, float mx) const {
        return (double)exp2f((float)((double)e - (double)mx * (double)c));
    }
    QMM_DEVINL bool fast(float mx, double T) const {
        return fabsf(mx) <= kFastMax && T >= kFastMinT && T <= kFastMaxT;
    }
};

// Sum of weights of one lane against its reference E.
struct LaneSum {
    float e = -3e38f;
    double s = 0.0;
};

// Such a sum against a larger reference, `by` the factor between them.  Tokens
// that are all masked with a huge number have a sum of any value, infinity among
// them, against their own E; by 0 it is nothing.  A NaN stays.
QMM_DEVINL double rescaled(double s, float by) { return by > 0.0f || s != s ? s * (double)by : 0.0; }

// In a tree: one long chain of 64-bit additions outlasts the weights themselves.
template <typename T, int N>
QMM_DEVINL T tree_sum(T (&e)[N]) {
#pragma unroll
    for (int h = N / 2; h >= 1; h /= 2)
#pragma unroll
        for (int j = 0; j < h; ++j) e[j] += e[j + h];
    return e[0];
}

// ---- a cluster's slices --------------------------------------------------------------

// The vectors of a warp.  Those from `begin` to `end` lie whole within the row,
// lane l takes begin + l, begin + l + 32, ..; the row's first and last vector,
// where they stick out of it, are `head` and `tail` (or -1) of the warp they
// fall to, and lane 0's.
struct Slice {
    int begin, end, head, tail;
    int lane;
};

template <int DT>
QMM_DEVINL Slice warp_slice(const Row<DT>& row, int warp, int warps) {
    const int per = (row.nv + warps - 1) / warps;
    const long long b = (long long)per * warp;
    Slice s;
    s.begin = (int)(b < row.nv ? b : row.nv);
    s.end = (int)(b + per < row.nv ? b + per : row.nv);
    s.lane = threadIdx.x & 31;
    s.head = s.tail = -1;
    if (s.begin < s.end && s.begin == 0 && !row.whole(0)) {
        s.head = 0;
        ++s.begin;
    }
    if (s.begin < s.end && s.end == row.nv && !row.whole(row.nv - 1)) s.tail = --s.end;
    return s;
}

// f(vectors, first index, how many) over the warp's slice: batches of 4 vectors
// 32 apart, the next batch's loads issued before f is called on this one.
template <int DT, typename F>
QMM_DEVINL void for_batches(const Row<DT>& row, const Slice& s, F&& f) {
    using Four = std::integral_constant<int, 4>;
    using One = std::integral_constant<int, 1>;
    int v = s.begin + s.lane;
    if (v + 96 < s.end) {
        uint4 next[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) next[i] = row.load_whole(v + 32 * i);
        do {
            uint4 u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = next[i];
            const int at = v;
            v += 128;
            if (v + 96 < s.end) {
#pragma unroll
                for (int i = 0; i < 4; ++i) next[i] = row.load_whole(v + 32 * i);
            }
            f(u, at, Four());
        } while (v + 96 < s.end);
    }
    if (v < s.end) {  // up to 4 more
        uint4 u[4];
        u[0] = row.load_whole(v);
#pragma unroll
        for (int i = 1; i < 4; ++i)
            if (v + 32 * i < s.end) u[i] = row.load_whole(v + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (v + 32 * i < s.end) f(&u[i], v + 32 * i, One());
    }
    if (s.lane == 0) {
        if (s.head >= 0) {
            uint4 u = row.load(s.head);
            f(&u, s.head, One());
        }
        if (s.tail >= 0) {
            uint4 u = row.load(s.tail);
            f(&u, s.tail, One());
        }
    }
}

// The same through shared memory, the next batch on its way all along: kStream
// slots of a thread.  For passes that also write (1024 gradient rows of 248320:
// 151 us, with registers for the batch ahead 173).
constexpr int kStages = 2, kStream = 4 * kStages;
using StreamRing = uint4 (*)[kRowThreads];  // [kStream][kRowThreads]

QMM_DEVINL void async_copy16(uint4* to, const void* from) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
}
QMM_DEVINL void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
QMM_DEVINL void async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int DT, typename F>
QMM_DEVINL void for_batches(const Row<DT>& row, const Slice& s, StreamRing ring, F&& f) {
    using Four = std::integral_constant<int, 4>;
    using One = std::integral_constant<int, 1>;
    const int t = threadIdx.x;
    auto issue = [&](int stage, int v) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (v + 32 * i < s.end) async_copy16(&ring[4 * stage + i][t], row.base + 16LL * (v + 32 * i));
        async_commit();
    };
    int v = s.begin + s.lane;
#pragma unroll
    for (int i = 0; i < kStages; ++i) issue(i, v + 128 * i);
    if (s.lane == 0) {
        if (s.head >= 0) {
            uint4 u = row.load(s.head);
            f(&u, s.head, One());
        }
        if (s.tail >= 0) {
            uint4 u = row.load(s.tail);
            f(&u, s.tail, One());
        }
    }
    int stage = 0;
#pragma unroll 1
    for (; v < s.end; v += 128) {
        async_wait<kStages - 1>();
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = ring[4 * stage + i][t];
        if (v + 96 < s.end) {
            f(u, v, Four());
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (v + 32 * i < s.end) f(&u[i], v + 32 * i, One());
        }
        issue(stage, v + 128 * kStages);
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    async_wait<0>();
}

// f(vector index, vector) over the warp's slice.
template <int DT, typename F, typename... R>
QMM_DEVINL void for_vectors(const Row<DT>& row, const Slice& s, F&& f, R... ring) {
    for_batches<DT>(row, s, ring..., [&](uint4* u, int v, auto n_) {
#pragma unroll
        for (int i = 0; i < decltype(n_)::value; ++i) f(v + 32 * i, u[i]);
    });
}

// The same in few instructions, for what hardly ever runs.
template <int DT, typename F>
QMM_DEVINL void for_vectors_rare(const Row<DT>& row, const Slice& s, F&& f) {
    const int first = s.head >= 0 ? s.head : s.begin, last = s.tail >= 0 ? s.tail + 1 : s.end;
#pragma unroll 1
    for (int v = first + s.lane; v < last; v += 32) f(v, row.load(v));
}

// The same for passes whose arithmetic in 64 bits needs the registers: vectors
// one at a time, the next three on their way into shared memory (cp.async, each
// thread's own slots, so nothing has to be synchronised).
constexpr int kRing = 4;
using Ring = uint4 (*)[kRowThreads];  // [kRing][kRowThreads] in shared memory

template <int DT, typename F>
QMM_DEVINL void for_vectors_slow(const Row<DT>& row, const Slice& s, Ring ring, F&& f) {
    const int t = threadIdx.x;
    int v = s.begin + s.lane;
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) {
        if (v + 32 * i < s.end) async_copy16(&ring[i][t], row.base + 16LL * (v + 32 * i));
        async_commit();
    }
    // the row's ends meanwhile
    if (s.lane == 0 && s.head >= 0) f(s.head, row.load(s.head));
    int slot = 0;
#pragma unroll 1
    for (; v < s.end; v += 32) {
        async_wait<kRing - 2>();
        const uint4 u = ring[slot][t];
        // into the slot that the round before has used up
        const int free = slot == 0 ? kRing - 1 : slot - 1, ahead = v + 32 * (kRing - 1);
        if (ahead < s.end) async_copy16(&ring[free][t], row.base + 16LL * ahead);
        async_commit();
        slot = slot == kRing - 1 ? 0 : slot + 1;
        f(v, u);
    }
    async_wait<0>();
    if (s.lane == 0 && s.tail >= 0) f(s.tail, row.load(s.tail));
}

// The two vectors of a lane with the largest maxima, these, and the largest of
// the lane's other vectors (or more, beside a NaN).
struct LaneTop {
    float first = kLow, second = kLow, others = kLow;
    int at = -1, at2 = -1;
    static constexpr float kLow = -__builtin_huge_valf();

    QMM_DEVINL void add(float m, int v) {
        const bool up = m > first, mid = m > second;
        others = fmaxf(others, fminf(m, second));
        second = up ? first : fmaxf(second, m);
        at2 = up ? at : mid ? v : at2;
        first = fmaxf(first, m);
        at = up ? v : at;
    }
};

// Maxima of the slice's logits in this lane (WHERE: and where they are), and
// with SUM the lane's weights.  change(vector index, vector) may take elements
// out (set them to -infinity).
template <int DT, bool SUM, bool WHERE, typename F, typename... R>
QMM_DEVINL LaneTop stream_slice(const Row<DT>& row, const Slice& s, const Scale& c, LaneSum& acc, F&& change,
                                R... ring) {
    constexpr int N = Elem<DT>::kVec;
    LaneTop top;
    for_batches<DT>(row, s, ring..., [&](uint4* u, int v, auto n_) {
        constexpr int n = decltype(n_)::value;
#pragma unroll
        for (int i = 0; i < n; ++i) change(v + 32 * i, u[i]);
        float bm = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float m = vec_max<DT>(u[i]);
            if (WHERE) top.add(m, v + 32 * i);
            bm = fmaxf(bm, m);
        }
        if (!WHERE) top.first = fmaxf(top.first, bm);
        if (!SUM) return;
        const float t = bm * c.c;
        if (t > acc.e + 16.0f) {  // weights stay below 2^17
            const float e = ceilf(t);
            acc.s = rescaled(acc.s, ex2(acc.e - e));
            acc.e = e;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            float e[N];
            decode<DT>(u[i], e);
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] = ex2(fmaf(e[j], c.c, -acc.e));
            sum += tree_sum(e);
        }
        acc.s += (double)sum;
    });
    return top;
}

template <int DT, bool SUM, bool WHERE>
QMM_DEVINL LaneTop stream_slice(const Row<DT>& row, const Slice& s, const Scale& c, LaneSum& acc) {
    return stream_slice<DT, SUM, WHERE>(row, s, c, acc, [](int, uint4&) {});
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

// What a warp knows of a row after its pass: the maximum, and the sum of
// weights against 2^e (without sums, e is the lowest of its lanes' maxima).
struct alignas(16) WarpStat {
    double s;
    float top, e;
};

QMM_DEVINL WarpStat warp_stat(float top, const LaneSum& acc, bool sum = true) {
    WarpStat w;
    w.top = warp_max(top);
    w.s = 0.0;
    if (!sum) {
        w.e = -warp_max(top == -CUDART_INF_F ? top : -top);
        return w;
    }
    w.e = warp_max(acc.e);
    w.s = warp_sum(rescaled(acc.s, ex2(acc.e - w.e)));
    return w;
}

// From the gathered warps: the row's maximum, its sum against the weight of the
// maximum (NaN where 32 bits do not do), and each warp's part of it into
// `slots` (by warp 0; null: not wanted).  Alike in every warp.
template <typename S>
QMM_DEVINL void row_stat(const WarpStat* stats, int warps, const S& c, float& mx, double& total, double* slots,
                         bool sum = true) {
    const int lane = threadIdx.x & 31;
    mx = -CUDART_INF_F;
    for (int i = lane; i < warps; i += 32) mx = fmaxf(mx, stats[i].top);
    mx = warp_max(mx);
    total = 0.0;
    if (!sum) return;
    const float e = ceilf(mx * c.c);
    const double back = c.against(e, mx);
    for (int i = lane; i < warps; i += 32) {
        const double x = rescaled(stats[i].s, ex2(stats[i].e - e)) * back;
        if (slots && threadIdx.x < 32) slots[i] = x;
        total += x;
    }
    total = warp_sum(total);
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

// Within the vectors [from, to): the first id at which base + the running sum
// of weights passes `target`, with the sums just before and after it; the last
// id of any weight if none does.  By a whole CTA: each thread sums a few
// neighbouring vectors, and the one whose sum holds the place goes through its
// own again.  weights(v, vector, w) fills a vector's weights in 64 bits, 0 for
// elements outside the row; its code stands here once, for both turns: what
// runs once a call costs its fetching.
struct Found {
    int id;
    double before, after;
};

struct FindShared {
    double sums[kRowWarps];
    Found found;
    int last;  // thread with the last weight
};

template <int DT, typename W>
QMM_DEVINL Found find_place(const Row<DT>& row, int from, int to, double base, double target, Ring ring,
                            FindShared& sh, W&& weights) {
    constexpr int N = Elem<DT>::kVec;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int per = (to - from + kRowThreads - 1) / kRowThreads;
    const int first = min(from + per * t, to), end = min(first + per, to);
    __syncthreads();
    if (t == 0) {
        sh.found = Found{-1, 0.0, 0.0};
        sh.last = -1;
    }
    // a thread's vectors, all at once
    for (int i = 0; i < kRing && first + i < end; ++i) {
        if (row.whole(first + i)) async_copy16(&ring[i][t], row.base + 16LL * (first + i));
        else ring[i][t] = row.load(first + i);
    }
    async_commit();
    async_wait<0>();
    double mass = 0.0, run = 0.0;
    bool done = false;
    for (int turn = 0; turn < 2; ++turn) {
        Found f{-1, 0.0, 0.0};
#pragma unroll 1
        for (int v = first; v < end; ++v) {
            double w[N];
            const int i = v - first;
            weights(v, i < kRing ? ring[i][t] : row.load(v), w);
            if (turn == 0) {
                mass += tree_sum(w);
                continue;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (w[j] > 0.0 && !done) {
                    f.id = row.first(v) + j;
                    f.before = run;
                    run += w[j];
                    f.after = run;
                    done = run > target;
                }
            }
        }
        if (turn == 1) {
            sh.found = f;
            break;
        }
        double incl = mass;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(~0u, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) sh.sums[warp] = incl;
        __syncthreads();
        run = __shfl_up_sync(~0u, incl, 1);  // not incl - mass, which loses what is small beside mass
        run = base + (lane == 0 ? 0.0 : run);
        for (int i = 0; i < warp; ++i) run += sh.sums[i];
        // the first thread that passes, or the last with a weight
        const bool passes = mass > 0.0 && run + mass > target;
        const int hit = __syncthreads_or(passes);
        if (mass > 0.0) atomicMax(&sh.last, hit ? (passes ? kRowThreads - t : -1) : t);
        __syncthreads();
        if (sh.last != (hit ? kRowThreads - t : t)) break;
    }
    __syncthreads();
    return sh.found;
}

template <int DT, typename W>
QMM_DEVINL Found find_in_slice(const Row<DT>& row, const Slice& s, double base, double target, Ring ring,
                               FindShared& sh, W&& weights) {
    return find_place<DT>(row, s.head >= 0 ? s.head : s.begin, s.tail >= 0 ? s.tail + 1 : s.end, base, target, ring,
                          sh, weights);
}

}  // namespace qmm

namespace qmm_host {

// CTAs to a row: so many that a lane holds at most `most` vectors; more, down to
// 8 vectors to a lane, while the call has no more than `ctas` of them (what runs
// at once, or several times that where a row's work is uneven), and down to 2
// while there is one to an SM at most.
int row_cluster(long long rows, long long V, int elem_bytes, int ctas, int most = 64);

bool pdl_enabled();                                                   // tma.cuh
int ensure_smem_limit(const void* func, int bytes, const char* what);  // tma.cuh

// Launch `kernel` over rows * C CTAs in clusters of C.  AFTER: it may start while
// the stream's previous kernel runs, and waits for it itself.
template <bool AFTER = false, typename... P, typename... A>
int launch_rows(void (*kernel)(P...), int threads, long long rows, int C, size_t smem, cudaStream_t st,
                const char* what, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * C));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (AFTER && pdl_enabled()) {
        at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    cudaError_t e = cudaSuccess;
    if (C > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && smem > 16 * 1024) {  // beside the kernel's static memory
        const int rc = ensure_smem_limit(reinterpret_cast<const void*>(kernel), (int)smem, what);
        if (rc) return rc;
    }
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return cuda_status(e, what);
}

}  // namespace qmm_host
