// logits_args.cuh -- one call of each operator on rows of logits, as the C
// entry points hand it to the kernels.  Strides count elements.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace qmm {

constexpr int kCand = 2048;     // candidates a row's cluster keeps: the largest k of a top-k is half of it
constexpr int kMaxList = 512;   // entries of a teacher's list

struct SampleArgs {
    const void* logits;
    long long stride;  // elements between rows
    int V;
    const float* u;
    // one value a row, or (null) one for all
    const float* t_rows;
    const int32_t* k_rows;
    const float* p_rows;
    const float* m_rows;
    double t, p, m;
    int k;
    int64_t* ids;
};

struct TopkArgs {
    const void* logits;
    long long stride;
    int V, k;
    double inv_t;
    void* values;
    int64_t* ids;
    float* lse;  // or null
};

struct RowStat {
    double sum;  // NaN: only a sum in 64 bits will do
    double inv_t;
    float mx;
    int arg;  // lowest id of the maximum, of greedy rows
};

struct SpecArgs {
    const void* logits;  // [B, n + 1, V]
    const void* draft;   // [B, n, V]
    long long stride_b, stride_i, dstride_b, dstride_i;
    int B, n, V;
    const int64_t* ids;  // [B, n]
    const float* u;      // [B, n + 1]
    const float* t_rows;   // [B] or null
    const float* dt_rows;  // likewise, of the draft
    double t, dt;
    RowStat* stats;  // [B, 2 n + 1]: the model's rows, then the draft's
    int64_t* tokens;
    int64_t* accepted;
};

enum { kLoss = 0, kLossGrad = 1, kBackward = 2 };

struct DistillArgs {
    const void* logits;
    long long stride;
    int V, k;
    const void* tv;
    int tv_dtype;
    const void* ti;
    int ti_bytes;
    const float* tlse;    // or null
    const float* weight;  // gradient's factor a row, or null (1)
    double inv_t;
    float* loss;    // not written by the backward pass
    float4* stats;  // (reference, factor of the others, maximum, sum) of a row: written by the loss, read by backward
    void* grad;
    long long grad_stride;
};

}  // namespace qmm

namespace qmm_host {
int launch_sample(const qmm::SampleArgs& a, long long rows, int dtype, cudaStream_t st);
int launch_topk(const qmm::TopkArgs& a, long long rows, int dtype, cudaStream_t st);
size_t speculative_workspace(long long B, long long n);
int launch_speculative(const qmm::SpecArgs& a, int dtype, cudaStream_t st);
int launch_distill(const qmm::DistillArgs& a, long long rows, int dtype, int mode, cudaStream_t st);
}  // namespace qmm_host
