// mx_capi.cu -- the C entry points of the microscaled formats
// (include/mlxturbo_b200.h): argument checks, workspace layout, kernel choice.

#include <initializer_list>

#include "mx.cuh"

namespace qmm_host {
size_t sort_workspace(long long M, long long E);
size_t route_smem(long long M, long long E);
bool sort_rows_takes(long long M, long long E);
int launch_moe_route(const uint32_t* ids, int M, int E, int top_k, int ir, uint32_t* order, uint32_t* idx_s,
                     uint32_t* row_src, uint32_t* inv, int32_t* row_start, int32_t* item_prefix, int4* item_info,
                     cudaStream_t st, const int32_t* lhs = nullptr);
int launch_sort_rows(const uint32_t* ids, long long rows, int E, int top_k, uint32_t* order, uint32_t* idx_s,
                     uint32_t* row_src, uint32_t* inv, void* ws, size_t ws_bytes, cudaStream_t st);
int launch_compose(const int32_t* lhs, const uint32_t* order, uint32_t* out, long long n, cudaStream_t st);
}  // namespace qmm_host

using namespace qmm_host;

namespace {

constexpr int64_t kMaxDim = 1LL << 30;

size_t al256(size_t b) { return (b + 255) & ~(size_t)255; }

// rows x K values in blocks of 32; rows * K stays an int64.
int check_rows(const char* what, int64_t rows, int64_t K) {
    if (rows < 0 || K <= 0 || K % qmm::MX_BLOCK) {
        set_error("%s: bad shape rows=%lld K=%lld (K must be a positive multiple of 32)", what, (long long)rows,
                  (long long)K);
        return QMM_EINVAL;
    }
    if (rows > kMaxDim || K > kMaxDim) {
        set_error("%s: rows=%lld K=%lld exceed the 2^30 limit", what, (long long)rows, (long long)K);
        return QMM_EUNSUPPORTED;
    }
    return QMM_OK;
}

int check_half(const char* what, int dtype) {
    if (dtype == QMM_BF16 || dtype == QMM_F16) return QMM_OK;
    set_error("%s: dtype %d must be bf16 or fp16", what, dtype);
    return QMM_EUNSUPPORTED;
}

int check_codec(const char* what, int bits, int dtype) {
    if (bits != 4 && bits != 8) {
        set_error("%s: bits=%d: the MX formats here have 4- and 8-bit codes", what, bits);
        return QMM_EUNSUPPORTED;
    }
    if (dtype != QMM_BF16 && dtype != QMM_F16 && dtype != QMM_F32) {
        set_error("%s: dtype %d must be bf16, fp16 or fp32", what, dtype);
        return QMM_EUNSUPPORTED;
    }
    return QMM_OK;
}

int check_aligned(const char* what, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (!p || !aligned16(p)) {
            set_error("%s: null pointer, or a tensor that is not 16-byte aligned", what);
            return QMM_EINVAL;
        }
    return QMM_OK;
}

int check_product(const char* what, int64_t M, int64_t N, int64_t K, int dtype) {
    int rc = check_half(what, dtype);
    if (rc) return rc;
    if ((rc = check_rows(what, M, K))) return rc;
    if (N <= 0) {
        set_error("%s: bad shape N=%lld", what, (long long)N);
        return QMM_EINVAL;
    }
    if (N > kMaxDim) {
        set_error("%s: N=%lld exceeds the 2^30 limit", what, (long long)N);
        return QMM_EUNSUPPORTED;
    }
    return QMM_OK;
}

// What the kernel for many rows can index.
int check_limits(const char* what, int64_t rows, int64_t E, int64_t N, int64_t K) {
    if (mx_tc_takes(rows, E, N, K)) return QMM_OK;
    set_error("%s: rows=%lld E=%lld N=%lld K=%lld beyond limits", what, (long long)rows, (long long)E, (long long)N,
              (long long)K);
    return QMM_EUNSUPPORTED;
}

int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
    if (need && (!ws || ((uintptr_t)ws & 255u) || have < need)) {
        set_error("%s: workspace must be 256-byte aligned and hold %zu bytes (%zu given)", what, need, have);
        return QMM_EINVAL;
    }
    return QMM_OK;
}

// Row tables of a grouped product, at the front of its workspace.
struct GatherTables {
    uint32_t *order, *idx_s, *row_src, *inv;  // unsorted ids only
    void* sort_ws;
    size_t sort_bytes;
    int32_t *row_start, *item_prefix, *n_items;
    int4* items;
    long long items_max;
    int item_rows;
    size_t bytes;
};

GatherTables gather_tables(void* base, int64_t rows, int64_t E, int sorted, int item_rows) {
    GatherTables t{};
    char* const p0 = static_cast<char*>(base);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* p = p0 + at;
        at += al256(bytes);
        return p;
    };
    t.item_rows = item_rows;
    t.items_max = rows / item_rows + (E < rows ? E : rows) + 1;
    t.row_start = reinterpret_cast<int32_t*>(take((size_t)(E + 1) * 4));
    t.item_prefix = reinterpret_cast<int32_t*>(take((size_t)(E + 1) * 4));
    t.n_items = reinterpret_cast<int32_t*>(take(4));
    t.items = reinterpret_cast<int4*>(take((size_t)t.items_max * sizeof(int4)));
    if (!sorted) {
        t.order = reinterpret_cast<uint32_t*>(take((size_t)rows * 4));
        t.idx_s = reinterpret_cast<uint32_t*>(take((size_t)rows * 4));
        t.row_src = reinterpret_cast<uint32_t*>(take((size_t)rows * 4));
        t.inv = reinterpret_cast<uint32_t*>(take((size_t)rows * 4));
        t.sort_bytes = sort_workspace(rows, E);
        t.sort_ws = take(t.sort_bytes);
    }
    t.bytes = at;
    return t;
}

}  // namespace

extern "C" {

int qmm_mx_quantize(const void* v, uint32_t* words, uint8_t* scales, int64_t rows, int64_t K, int bits, int dtype,
                    void* stream) {
    clear_error();
    int rc = check_codec("mx_quantize", bits, dtype);
    if (rc) return rc;
    if ((rc = check_rows("mx_quantize", rows, K))) return rc;
    if (rows == 0) return QMM_OK;
    if ((rc = check_aligned("mx_quantize", {v, words}))) return rc;
    if (!scales) {
        set_error("mx_quantize: null pointer");
        return QMM_EINVAL;
    }
    fire("mx_quantize");
    return launch_mx_quantize(v, words, scales, rows * K, bits, dtype, static_cast<cudaStream_t>(stream));
}

int qmm_mx_dequantize(const uint32_t* words, const uint8_t* scales, void* out, int64_t rows, int64_t K, int bits,
                      int dtype, void* stream) {
    clear_error();
    int rc = check_codec("mx_dequantize", bits, dtype);
    if (rc) return rc;
    if ((rc = check_rows("mx_dequantize", rows, K))) return rc;
    if (rows == 0) return QMM_OK;
    if ((rc = check_aligned("mx_dequantize", {words, out}))) return rc;
    if (!scales) {
        set_error("mx_dequantize: null pointer");
        return QMM_EINVAL;
    }
    fire("mx_dequantize");
    return launch_mx_dequantize(words, scales, out, rows * K, bits, dtype, static_cast<cudaStream_t>(stream));
}

int qmm_mx_rms_norm(const void* x, const void* residual, const void* weight, void* h, uint32_t* xq,
                    uint8_t* x_scales, int64_t rows, int64_t K, float eps, int dtype, void* stream) {
    clear_error();
    int rc = check_half("mx_rms_norm", dtype);
    if (rc) return rc;
    if ((rc = check_rows("mx_rms_norm", rows, K))) return rc;
    if (!(eps >= 0.0f)) {
        set_error("mx_rms_norm: eps must not be negative");
        return QMM_EINVAL;
    }
    if (rows == 0) return QMM_OK;
    if ((rc = check_aligned("mx_rms_norm", {x, weight, xq}))) return rc;
    if (residual && (rc = check_aligned("mx_rms_norm", {residual, h}))) return rc;
    if (!x_scales || (residual && (h == x || h == residual))) {
        set_error("mx_rms_norm: null pointer, or h is x or residual");
        return QMM_EINVAL;
    }
    fire("mx_rms_norm");
    return launch_mx_rms_norm(x, residual, weight, h, xq, x_scales, rows, K, eps, dtype == QMM_F16,
                              static_cast<cudaStream_t>(stream));
}

size_t qmm_mx_matmul_workspace_size(int64_t M, int64_t N, int64_t K, int dtype, int x_is_mx) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 32) return 0;
    const int f4 = mx_f4_takes(M, 1, N, K, x_is_mx, false) ? mx_f4_item_rows(M, 1, N, K, x_is_mx, false) : 0;
    if (f4) return mx_f4_workspace(M, K, f4);
    return mx_tc_workspace(M, N, K, x_is_mx, dtype == QMM_F16, false);
}

int qmm_mx_matmul(const void* x, const uint8_t* x_scales, const uint32_t* w, const uint8_t* scales, void* y,
                  int64_t M, int64_t N, int64_t K, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_product("mx_matmul", M, N, K, dtype);
    if (rc) return rc;
    const bool mx = x_scales != nullptr;
    const int f4 = mx_f4_takes(M, 1, N, K, mx, false) ? mx_f4_item_rows(M, 1, N, K, mx, false) : 0;
    if (!f4 && (rc = check_limits("mx_matmul", M, 1, N, K))) return rc;
    if (M == 0) return QMM_OK;
    if ((rc = check_aligned("mx_matmul", {x, w, y}))) return rc;
    if (!scales) {
        set_error("mx_matmul: null pointer");
        return QMM_EINVAL;
    }
    if ((rc = check_workspace("mx_matmul", workspace, workspace_bytes,
                              qmm_mx_matmul_workspace_size(M, N, K, dtype, x_scales != nullptr))))
        return rc;
    MxMatmul a{};
    a.x = x;
    a.xs = x_scales;
    a.w = w;
    a.ws = scales;
    a.y = y;
    a.rows = a.x_rows = M;
    a.E = 1;
    a.N = N;
    a.K = K;
    a.f16 = dtype == QMM_F16;
    a.st = static_cast<cudaStream_t>(stream);
    fire("mx_matmul");
    if (f4) return launch_mx_f4(a, nullptr, nullptr, nullptr, f4, workspace);
    return launch_mx_tc(a, nullptr, nullptr, nullptr, workspace);
}

size_t qmm_mx_gather_workspace_size(int64_t rows, int64_t E, int64_t N, int64_t K, int dtype, int x_is_mx,
                                    int sorted) {
    if (rows <= 0 || E <= 0) return 0;
    if (K <= 0 || K % 32) return 0;
    const int f4 = mx_f4_takes(rows, E, N, K, x_is_mx, true) ? mx_f4_item_rows(rows, E, N, K, x_is_mx, true) : 0;
    if (f4) return gather_tables(nullptr, rows, E, sorted, f4).bytes + mx_f4_workspace(rows, K, f4);
    return gather_tables(nullptr, rows, E, sorted, mx_tc_item_rows()).bytes +
           mx_tc_workspace(rows, N, K, x_is_mx, dtype == QMM_F16, true);
}

int qmm_mx_gather(const void* x, const uint8_t* x_scales, const uint32_t* w, const uint8_t* scales,
                  const int32_t* lhs, const int32_t* rhs, void* y, int64_t rows, int64_t x_rows, int64_t E, int64_t N,
                  int64_t K, int dtype, int sorted, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_product("mx_gather", rows, N, K, dtype);
    if (rc) return rc;
    if (E <= 0 || x_rows < 0 || (rows > 0 && x_rows == 0) || (!lhs && x_rows < rows)) {
        set_error("mx_gather: bad shape rows=%lld x_rows=%lld E=%lld", (long long)rows, (long long)x_rows,
                  (long long)E);
        return QMM_EINVAL;
    }
    if (E > 16384 || x_rows > kMaxDim || (!sorted && !route_smem(rows, E) && !sort_rows_takes(rows, E))) {
        set_error("mx_gather: rows=%lld E=%lld x_rows=%lld beyond limits", (long long)rows, (long long)E,
                  (long long)x_rows);
        return QMM_EUNSUPPORTED;
    }
    const bool f16 = dtype == QMM_F16, mx = x_scales != nullptr;
    const int f4 = mx_f4_takes(rows, E, N, K, mx, true) ? mx_f4_item_rows(rows, E, N, K, mx, true) : 0;
    if (!f4 && (rc = check_limits("mx_gather", rows, E, N, K))) return rc;
    if (rows == 0) return QMM_OK;
    if ((rc = check_aligned("mx_gather", {x, w, y}))) return rc;
    if (!scales || !rhs) {
        set_error("mx_gather: null pointer");
        return QMM_EINVAL;
    }
    if ((rc = check_workspace("mx_gather", workspace, workspace_bytes,
                              qmm_mx_gather_workspace_size(rows, E, N, K, dtype, x_scales != nullptr, sorted))))
        return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int item_rows = f4 ? f4 : mx_tc_item_rows();
    const GatherTables t = gather_tables(workspace, rows, E, sorted, item_rows);
    MxMatmul a{};
    a.x = x;
    a.xs = x_scales;
    a.w = w;
    a.ws = scales;
    a.y = y;
    a.rows = rows;
    a.x_rows = x_rows;
    a.E = E;
    a.N = N;
    a.K = K;
    a.f16 = f16;
    a.st = st;
    const int32_t* n_items = t.n_items;
    if (f4 && mx_f4_direct(rows, E, true)) {
        fire("mx_gather");
        a.lhs = lhs;
        return launch_mx_f4(a, nullptr, nullptr, rhs, f4, nullptr);
    }
    if (sorted) {
        rc = launch_mx_items(rhs, rows, (int)E, t.item_rows, t.row_start, t.items, t.items_max, t.n_items, st);
        a.src = reinterpret_cast<const uint32_t*>(lhs);
    } else {
        if (route_smem(rows, E)) {  // a decode batch: sort, tables and x rows in one launch
            rc = launch_moe_route(reinterpret_cast<const uint32_t*>(rhs), (int)rows, (int)E, 1, t.item_rows, t.order,
                                  t.idx_s, t.row_src, t.inv, t.row_start, t.item_prefix, t.items, st, lhs);
            n_items = t.item_prefix + E;
        } else {
            rc = launch_sort_rows(reinterpret_cast<const uint32_t*>(rhs), rows, (int)E, 1, t.order, t.idx_s, t.row_src,
                                  t.inv, t.sort_ws, t.sort_bytes, st);
            if (!rc)
                rc = launch_mx_items(reinterpret_cast<const int32_t*>(t.idx_s), rows, (int)E, t.item_rows, t.row_start,
                                     t.items, t.items_max, t.n_items, st);
            if (!rc && lhs) rc = launch_compose(lhs, t.order, t.row_src, rows, st);
        }
        a.dst = t.order;
        a.src = t.row_src;
    }
    if (rc) return rc;
    fire("mx_gather");
    if (f4) return launch_mx_f4(a, t.items, n_items, rhs, f4, static_cast<char*>(workspace) + t.bytes);
    return launch_mx_tc(a, t.items, n_items, rhs, static_cast<char*>(workspace) + t.bytes);
}

}  // extern "C"
