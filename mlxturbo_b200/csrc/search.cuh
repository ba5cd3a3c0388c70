// search.cuh -- searches for a border with a bound on their steps.  They hold
// for any values: float keys lie far denser around 0 than weights tell apart,
// so a border may be 1e9 keys from where its formula puts it.  Compiles for the
// host too, where its tests run.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define QMM_SEARCH __host__ __device__ __forceinline__
#else
#define QMM_SEARCH inline
#endif

namespace qmm {

// The lowest key of [lo, hi] from which on up to hi all are kept; hi is.  Strides
// that double lead from the guess past the border, a bisection back to it: two
// calls of keeps() where the guess is right, 66 at most.
template <typename F>
QMM_SEARCH uint32_t lowest_kept(uint32_t lo, uint32_t hi, uint32_t guess, F&& keeps) {
    uint32_t in = guess < lo ? lo : guess < hi ? guess : hi, out, stride = 1;
    if (in == hi || keeps(in)) {
        for (;;) {
            if (in == lo) return lo;
            const uint32_t at = in - lo > stride ? in - stride : lo;
            if (!keeps(at)) {
                out = at;
                break;
            }
            in = at;
            if (stride < 0x80000000u) stride *= 2;
        }
    } else {
        out = in;
        for (;;) {
            in = hi - out > stride ? out + stride : hi;
            if (in == hi || keeps(in)) break;
            out = in;
            if (stride < 0x80000000u) stride *= 2;
        }
    }
    while (in - out > 1) {
        const uint32_t mid = out + (in - out) / 2;
        if (keeps(mid)) in = mid;
        else out = mid;
    }
    return in;
}

}  // namespace qmm
