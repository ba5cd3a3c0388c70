// logits_capi.cu -- the C entry points of the operators on rows of logits
// (include/mlxturbo_b200.h): argument checks.

#include <math.h>

#include "logits_args.cuh"

using namespace qmm_host;

namespace {

constexpr int64_t kMaxVocab = 1LL << 30;  // ids and vector counts are ints
constexpr int64_t kMaxRows = 1LL << 26;   // rows * 16 CTAs in one grid
constexpr int64_t kMaxDraft = 1LL << 16;  // a warp looks through a sequence's ids before each of its rows

int check_rows(const char* what, int64_t rows, int64_t V, int64_t stride, int dtype) {
    if (dtype != QMM_BF16 && dtype != QMM_F16 && dtype != QMM_F32) {
        set_error("%s: dtype %d must be bf16, fp16 or fp32", what, dtype);
        return QMM_EUNSUPPORTED;
    }
    if (rows < 0 || V <= 0 || stride < 0) {
        set_error("%s: bad shape rows=%lld V=%lld row stride %lld", what, (long long)rows, (long long)V,
                  (long long)stride);
        return QMM_EINVAL;
    }
    if (rows > kMaxRows || V > kMaxVocab) {
        set_error("%s: rows=%lld V=%lld exceed the limits 2^26 and 2^30", what, (long long)rows, (long long)V);
        return QMM_EUNSUPPORTED;
    }
    return QMM_OK;
}

// Logits start at any element; other arrays at theirs.
bool askew(const void* p, int bytes) { return (uintptr_t)p % bytes; }  // null, an array that is not given, is not
bool misaligned(const void* p, int bytes) { return !p || askew(p, bytes); }

int check_temperature(const char* what, double t, bool zero) {
    if (zero && t == 0.0) return QMM_OK;
    if (t >= 1e-6 && t <= 1e6) return QMM_OK;
    set_error("%s: temperature %g is not in [1e-6, 1e6]%s", what, t, zero ? " and not 0" : "");
    return QMM_EINVAL;
}

int elem_bytes(int dtype) { return dtype == QMM_F32 ? 4 : 2; }

int null_error(const char* what) {
    set_error("%s: null or misaligned pointer", what);
    return QMM_EINVAL;
}

int distill_args(const char* what, qmm::DistillArgs& d, const void* logits, int64_t row_stride, int64_t rows,
                 int64_t V, int dtype, const void* teacher_values, int teacher_dtype, const void* teacher_ids,
                 int id_bytes, const float* teacher_logsumexp, int64_t k, double temperature) {
    int rc = check_rows(what, rows, V, row_stride, dtype);
    if (rc) return rc;
    if ((rc = check_temperature(what, temperature, false))) return rc;
    if (teacher_dtype != QMM_BF16 && teacher_dtype != QMM_F16 && teacher_dtype != QMM_F32) {
        set_error("%s: teacher dtype %d must be bf16, fp16 or fp32", what, teacher_dtype);
        return QMM_EUNSUPPORTED;
    }
    if (k < 1 || (id_bytes != 4 && id_bytes != 8)) {
        set_error("%s: k=%lld must be positive, ids of 4 or 8 bytes (%d)", what, (long long)k, id_bytes);
        return QMM_EINVAL;
    }
    if (k > qmm::kMaxList) {
        set_error("%s: k=%lld exceeds the limit %d", what, (long long)k, qmm::kMaxList);
        return QMM_EUNSUPPORTED;
    }
    if (rows && (misaligned(logits, elem_bytes(dtype)) || misaligned(teacher_values, elem_bytes(teacher_dtype)) ||
                 misaligned(teacher_ids, id_bytes) || askew(teacher_logsumexp, 4)))
        return null_error(what);
    d.logits = logits;
    d.stride = row_stride;
    d.V = (int)V;
    d.k = (int)k;
    d.tv = teacher_values;
    d.tv_dtype = teacher_dtype;
    d.ti = teacher_ids;
    d.ti_bytes = id_bytes;
    d.tlse = teacher_logsumexp;
    d.inv_t = 1.0 / temperature;
    return QMM_OK;
}

}  // namespace

extern "C" {

int qmm_sample(const void* logits, int64_t row_stride, int64_t rows, int64_t V, int dtype, const float* u,
               const float* temperature_rows, double temperature, const int32_t* top_k_rows, int64_t top_k,
               const float* top_p_rows, double top_p, const float* min_p_rows, double min_p, int64_t* ids,
               void* stream) {
    clear_error();
    int rc = check_rows("sample", rows, V, row_stride, dtype);
    if (rc) return rc;
    if (!temperature_rows && (rc = check_temperature("sample", temperature, true))) return rc;
    if (!top_k_rows && top_k < 0) {
        set_error("sample: top_k=%lld must not be negative (0 keeps all)", (long long)top_k);
        return QMM_EINVAL;
    }
    if (!top_p_rows && !(top_p > 0.0 && top_p <= 1.0)) {
        set_error("sample: top_p=%g is not in (0, 1]", top_p);
        return QMM_EINVAL;
    }
    if (!min_p_rows && !(min_p >= 0.0 && min_p <= 1.0)) {
        set_error("sample: min_p=%g is not in [0, 1]", min_p);
        return QMM_EINVAL;
    }
    if (rows == 0) return QMM_OK;
    if (misaligned(logits, elem_bytes(dtype)) || misaligned(u, 4) || misaligned(ids, 8) ||
        askew(temperature_rows, 4) || askew(top_k_rows, 4) || askew(top_p_rows, 4) || askew(min_p_rows, 4))
        return null_error("sample");
    qmm::SampleArgs a{};
    a.logits = logits;
    a.stride = row_stride;
    a.V = (int)V;
    a.u = u;
    a.t_rows = temperature_rows;
    a.k_rows = top_k_rows;
    a.p_rows = top_p_rows;
    a.m_rows = min_p_rows;
    a.t = temperature;
    a.p = top_p;
    a.m = min_p;
    a.k = (int)(top_k < V ? top_k : 0);
    a.ids = ids;
    fire("sample");
    return launch_sample(a, rows, dtype, static_cast<cudaStream_t>(stream));
}

int qmm_topk(const void* logits, int64_t row_stride, int64_t rows, int64_t V, int dtype, int64_t k,
             double temperature, void* values, int64_t* ids, float* logsumexp, void* stream) {
    clear_error();
    int rc = check_rows("topk", rows, V, row_stride, dtype);
    if (rc) return rc;
    if ((rc = check_temperature("topk", temperature, false))) return rc;
    if (k < 1 || k > V) {
        set_error("topk: k=%lld is not in [1, V=%lld]", (long long)k, (long long)V);
        return QMM_EINVAL;
    }
    if (k > qmm::kCand / 2) {
        set_error("topk: k=%lld exceeds the limit %d", (long long)k, qmm::kCand / 2);
        return QMM_EUNSUPPORTED;
    }
    if (rows == 0) return QMM_OK;
    if (misaligned(logits, elem_bytes(dtype)) || misaligned(values, elem_bytes(dtype)) || misaligned(ids, 8) ||
        askew(logsumexp, 4))
        return null_error("topk");
    qmm::TopkArgs a{};
    a.logits = logits;
    a.stride = row_stride;
    a.V = (int)V;
    a.k = (int)k;
    a.inv_t = 1.0 / temperature;
    a.values = values;
    a.ids = ids;
    a.lse = logsumexp;
    fire("topk");
    return launch_topk(a, rows, dtype, static_cast<cudaStream_t>(stream));
}

size_t qmm_speculative_sample_workspace_size(int64_t B, int64_t n) {
    return B > 0 && n >= 0 && B <= kMaxRows && n <= kMaxRows ? speculative_workspace(B, n) : 0;
}

int qmm_speculative_sample(const void* logits, int64_t seq_stride, int64_t row_stride, const void* draft_logits,
                           int64_t draft_seq_stride, int64_t draft_row_stride, int64_t B, int64_t n, int64_t V,
                           int dtype, const int64_t* draft_ids, const float* u, const float* temperature_rows,
                           double temperature, const float* draft_temperature_rows, double draft_temperature,
                           int64_t* tokens, int64_t* accepted, void* workspace, size_t workspace_bytes,
                           void* stream) {
    clear_error();
    int rc = check_rows("speculative_sample", B, V, row_stride, dtype);
    if (rc) return rc;
    if (n < 0 || seq_stride < 0 || draft_seq_stride < 0 || draft_row_stride < 0) {
        set_error("speculative_sample: bad shape n=%lld or a negative stride", (long long)n);
        return QMM_EINVAL;
    }
    if (n > kMaxDraft || B * (2 * n + 1) > kMaxRows) {
        set_error("speculative_sample: B=%lld n=%lld exceed the limits of 2^16 drafted tokens and 2^26 rows",
                  (long long)B, (long long)n);
        return QMM_EUNSUPPORTED;
    }
    if (!temperature_rows && (rc = check_temperature("speculative_sample", temperature, true))) return rc;
    if (!draft_temperature_rows && (rc = check_temperature("speculative_sample", draft_temperature, true))) return rc;
    if (B == 0) return QMM_OK;
    if (misaligned(logits, elem_bytes(dtype)) || misaligned(u, 4) || misaligned(tokens, 8) || misaligned(accepted, 8) ||
        askew(temperature_rows, 4) || askew(draft_temperature_rows, 4) ||
        (n && (misaligned(draft_logits, elem_bytes(dtype)) || misaligned(draft_ids, 8))))
        return null_error("speculative_sample");
    const size_t need = speculative_workspace(B, n);
    if (misaligned(workspace, 16) || workspace_bytes < need) {
        set_error("speculative_sample: workspace must be 16-byte aligned and hold %zu bytes (%zu given)", need,
                  workspace_bytes);
        return QMM_EINVAL;
    }
    qmm::SpecArgs a{};
    a.logits = logits;
    a.draft = draft_logits;
    a.stride_b = seq_stride;
    a.stride_i = row_stride;
    a.dstride_b = draft_seq_stride;
    a.dstride_i = draft_row_stride;
    a.B = (int)B;
    a.n = (int)n;
    a.V = (int)V;
    a.ids = draft_ids;
    a.u = u;
    a.t_rows = temperature_rows;
    a.dt_rows = draft_temperature_rows;
    a.t = temperature;
    a.dt = draft_temperature;
    a.stats = static_cast<qmm::RowStat*>(workspace);
    a.tokens = tokens;
    a.accepted = accepted;
    fire("speculative");
    return launch_speculative(a, dtype, static_cast<cudaStream_t>(stream));
}

int qmm_distill_loss(const void* logits, int64_t row_stride, int64_t rows, int64_t V, int dtype,
                     const void* teacher_values, int teacher_dtype, const void* teacher_ids, int id_bytes,
                     const float* teacher_logsumexp, int64_t k, double temperature, float* loss, void* stats,
                     void* stream) {
    clear_error();
    qmm::DistillArgs d{};
    int rc = distill_args("distill_loss", d, logits, row_stride, rows, V, dtype, teacher_values, teacher_dtype,
                          teacher_ids, id_bytes, teacher_logsumexp, k, temperature);
    if (rc || rows == 0) return rc;
    if (misaligned(loss, 4) || askew(stats, 16)) return null_error("distill_loss");
    d.loss = loss;
    d.stats = static_cast<float4*>(stats);
    fire("distill_loss");
    return launch_distill(d, rows, dtype, qmm::kLoss, static_cast<cudaStream_t>(stream));
}

int qmm_distill_loss_grad(const void* logits, int64_t row_stride, int64_t rows, int64_t V, int dtype,
                          const void* teacher_values, int teacher_dtype, const void* teacher_ids, int id_bytes,
                          const float* teacher_logsumexp, int64_t k, double temperature, const float* row_weight,
                          float* loss, void* grad, int64_t grad_stride, void* stream) {
    clear_error();
    qmm::DistillArgs d{};
    int rc = distill_args("distill_loss_grad", d, logits, row_stride, rows, V, dtype, teacher_values, teacher_dtype,
                          teacher_ids, id_bytes, teacher_logsumexp, k, temperature);
    if (rc || rows == 0) return rc;
    if (misaligned(loss, 4) || misaligned(grad, elem_bytes(dtype)) || askew(row_weight, 4))
        return null_error("distill_loss_grad");
    if (grad_stride < V || (grad == logits && grad_stride != row_stride && rows > 1)) {
        set_error("distill_loss_grad: gradient rows %lld apart for V=%lld, logits %lld", (long long)grad_stride,
                  (long long)V, (long long)row_stride);
        return QMM_EINVAL;
    }
    d.weight = row_weight;
    d.loss = loss;
    d.grad = grad;
    d.grad_stride = grad_stride;
    fire("distill_grad");
    return launch_distill(d, rows, dtype, qmm::kLossGrad, static_cast<cudaStream_t>(stream));
}

int qmm_distill_backward(const void* logits, int64_t row_stride, int64_t rows, int64_t V, int dtype,
                         const void* teacher_values, int teacher_dtype, const void* teacher_ids, int id_bytes,
                         const float* teacher_logsumexp, int64_t k, double temperature, const void* stats,
                         const float* grad_loss, void* grad, int64_t grad_stride, void* stream) {
    clear_error();
    qmm::DistillArgs d{};
    int rc = distill_args("distill_backward", d, logits, row_stride, rows, V, dtype, teacher_values, teacher_dtype,
                          teacher_ids, id_bytes, teacher_logsumexp, k, temperature);
    if (rc || rows == 0) return rc;
    if (misaligned(stats, 16) || misaligned(grad_loss, 4) || misaligned(grad, elem_bytes(dtype)))
        return null_error("distill_backward");
    if (grad_stride < V || grad == logits) {
        set_error("distill_backward: the gradient must not be the logits, its rows %lld apart hold V=%lld",
                  (long long)grad_stride, (long long)V);
        return QMM_EINVAL;
    }
    d.weight = grad_loss;
    d.stats = static_cast<float4*>(const_cast<void*>(stats));
    d.grad = grad;
    d.grad_stride = grad_stride;
    fire("distill_grad");
    return launch_distill(d, rows, dtype, qmm::kBackward, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
