// torch_ops.cpp -- the public ops as PyTorch custom operators
// (torch.ops.mlxturbo_b200.*) over the C ABI of libmlxturbo_b200.so.
//
// A decode step makes one call per projection, and a projection runs for
// 4-14 us on the device, so the host time of a call bounds the end-to-end
// rate.  Through ctypes a call costs ~10 us (argument conversion, the stream
// handle, the workspace look-up, Python-side checks).  These operators do the
// same work in C++ behind the PyTorch dispatcher: the checks, the tensors'
// device pointers, the current CUDA stream, and one zeroed device workspace
// per device kept here (sized on demand; the decode kernels leave its counter
// block zero and tag their partial sums with a per-call epoch, exactly as with
// the Python layer's workspace).
//
// Signatures follow mx.quantized_matmul (mlxturbo/kernels/dispatch.py:317-327)
// with transpose=True, mode="affine"; an `out` tensor of the result shape may
// be given to reuse the output buffer.  Argument errors raise ValueError (a
// CPU tensor among the arguments included), unsupported dtypes / shapes
// NotImplementedError, with the library's message.  ops.quantized_matmul
// calls these directly and leaves every check to them.

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>
#include <torch/types.h>

#include <cstdarg>
#include <cstdio>
#include <initializer_list>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_map>

#include "../../include/mlxturbo_b200.h"

namespace {

// Error messages are formatted here with vsnprintf and handed to the check
// macros as one string: a message built by the macros' own stream formatting
// from several arguments (numbers, sizes) crashed the process (SIGSEGV) in
// this extension build, while a single string argument raises cleanly.
enum class Err { kValue, kNotImplemented, kRuntime };

[[noreturn]] void fail(Err kind, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    const char* m = buf;
    if (kind == Err::kValue) TORCH_CHECK_VALUE(false, m);
    if (kind == Err::kNotImplemented) TORCH_CHECK_NOT_IMPLEMENTED(false, m);
    TORCH_CHECK(false, m);
    __builtin_unreachable();
}

std::string dims(at::IntArrayRef d) {
    std::string r = "(";
    for (size_t i = 0; i < d.size(); ++i) {
        char b[32];
        std::snprintf(b, sizeof b, i ? ", %lld" : "%lld", (long long)d[i]);
        r += b;
    }
    return r + ")";
}

int dtype_code(const at::Tensor& x) {
    if (x.scalar_type() == at::kBFloat16) return QMM_BF16;
    if (x.scalar_type() == at::kHalf) return QMM_F16;
    fail(Err::kNotImplemented, "activations must be bfloat16 or float16, got %s", c10::toString(x.scalar_type()));
}

void check(int rc, const char* what) {
    if (rc == QMM_OK) return;
    const Err kind = rc == QMM_EUNSUPPORTED ? Err::kNotImplemented : rc == QMM_EINVAL ? Err::kValue : Err::kRuntime;
    fail(kind, "%s: %s: %s", what, qmm_status_string(rc), qmm_last_error());
}

// A zeroed uint8 buffer of at least `bytes` on `device`, kept for the process.
// Growing it replaces the buffer (the old one is released in stream order by
// the caching allocator); a new buffer starts at zero, as the kernels need.
at::Tensor& decode_workspace(const at::Device& device, size_t bytes) {
    static std::mutex mu;
    static std::unordered_map<int, at::Tensor> bufs;
    std::lock_guard<std::mutex> lock(mu);
    at::Tensor& buf = bufs[device.index()];
    if (!buf.defined() || (size_t)buf.numel() < bytes) {
        size_t size = 1u << 20;
        while (size < bytes) size <<= 1;
        buf = at::zeros({(int64_t)size}, at::TensorOptions().dtype(at::kByte).device(device));
    }
    return buf;
}

// A new tensor on the device of `like`, allocated without another pass through
// the dispatcher (about 0.3 us each: a norm and a dequantisation, four tensors,
// take 14.0 us of host time, with at::empty 14.9).
at::Tensor empty_like_device(at::IntArrayRef shape, at::ScalarType dtype, const at::Tensor& like) {
    return at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt);
}

at::Tensor contiguous16(const at::Tensor& t) {
    at::Tensor c = t.contiguous();
    if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16) c = c.clone();
    return c;
}

at::Tensor run_quantized_matmul(const at::Tensor& x_in, const at::Tensor& w_in, const at::Tensor& scales_in,
                                const at::Tensor& biases_in, int64_t group_size, int64_t bits,
                                const at::Tensor* out) {
    if (!(x_in.is_cuda() && w_in.is_cuda() && scales_in.is_cuda() && biases_in.is_cuda()))
        fail(Err::kValue, "mlxturbo_b200 ops take CUDA tensors (there is no CPU path)");
    if (!(w_in.device() == x_in.device() && scales_in.device() == x_in.device() &&
          biases_in.device() == x_in.device() && (!out || out->device() == x_in.device())))
        fail(Err::kValue, "x, w, scales, biases and out must be on one device");
    if (x_in.dim() < 1) fail(Err::kValue, "x must have at least one dimension");
    const int dt = dtype_code(x_in);
    const at::Tensor x = contiguous16(x_in), w = contiguous16(w_in);
    const at::Tensor s = scales_in.contiguous(), b = biases_in.contiguous();
    if (s.scalar_type() != x.scalar_type() || b.scalar_type() != x.scalar_type())
        fail(Err::kValue, "scales and biases must have the activations' dtype");
    const int64_t K = x.size(-1), N = w.dim() == 2 ? w.size(0) : -1, M = K ? x.numel() / K : 0;
    if (!(w.dim() == 2 && w.size(1) * 32 == K * bits))
        fail(Err::kValue, "w shape %s does not match K=%lld bits=%lld", dims(w.sizes()).c_str(), (long long)K,
             (long long)bits);
    if (!(group_size > 0 && K % group_size == 0 && s.dim() == 2 && s.size(0) == N && s.size(1) == K / group_size &&
          b.sizes() == s.sizes()))
        fail(Err::kValue, "scales/biases shape %s != (%lld, %lld)", dims(s.sizes()).c_str(), (long long)N,
             (long long)(K / (group_size > 0 ? group_size : 1)));
    c10::cuda::CUDAGuard guard(x.device());
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    at::Tensor y;
    if (out) {
        y = *out;
        if (!(y.is_contiguous() && y.sizes() == at::IntArrayRef(shape) && y.scalar_type() == x.scalar_type() &&
              reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0))
            fail(Err::kValue, "out must be a contiguous, 16-byte aligned tensor of the result shape %s and x's dtype",
                 dims(at::IntArrayRef(shape)).c_str());
    } else {
        y = at::empty(shape, x.options());
    }
    if (M == 0) return y;
    const size_t need = qmm_quantized_matmul_workspace_size(M, N, K, (int)group_size, (int)bits);
    void* ws = nullptr;
    size_t ws_bytes = 0;
    if (need) {
        at::Tensor& buf = decode_workspace(x.device(), need);
        ws = buf.data_ptr();
        ws_bytes = (size_t)buf.numel();
    }
    const cudaStream_t st = at::cuda::getCurrentCUDAStream(x.device().index()).stream();
    check(qmm_quantized_matmul(x.data_ptr(), static_cast<const uint32_t*>(w.data_ptr()), s.data_ptr(), b.data_ptr(),
                               y.data_ptr(), M, N, K, (int)group_size, (int)bits, dt, ws, ws_bytes, st),
          "quantized_matmul");
    return y;
}

at::Tensor quantized_matmul(const at::Tensor& x, const at::Tensor& w, const at::Tensor& scales,
                            const at::Tensor& biases, int64_t group_size, int64_t bits) {
    return run_quantized_matmul(x, w, scales, biases, group_size, bits, nullptr);
}

at::Tensor& quantized_matmul_out(const at::Tensor& x, const at::Tensor& w, const at::Tensor& scales,
                                 const at::Tensor& biases, int64_t group_size, int64_t bits, at::Tensor& out) {
    run_quantized_matmul(x, w, scales, biases, group_size, bits, &out);
    return out;
}

// ---- microscaled (MX) formats -----------------------------------------------
// Words are 4-byte integers (int32 or uint32), scales one byte each (uint8).
// Scratch comes from the caching allocator per call (the kernels ask nothing of
// its content), so calls on different streams do not share any.

int mx_dtype_code(at::ScalarType t) {
    if (t == at::kBFloat16) return QMM_BF16;
    if (t == at::kHalf) return QMM_F16;
    if (t == at::kFloat) return QMM_F32;
    fail(Err::kNotImplemented, "dtype must be bfloat16, float16 or float32, got %s", c10::toString(t));
}

int mx_half_code(at::ScalarType t) {
    if (t == at::kFloat) fail(Err::kNotImplemented, "dtype must be bfloat16 or float16, got %s", c10::toString(t));
    return mx_dtype_code(t);
}

void mx_same_device(const char* what, std::initializer_list<const at::Tensor*> ts) {
    const at::Tensor* first = nullptr;
    for (const at::Tensor* t : ts) {
        if (!t) continue;
        if (!t->is_cuda()) fail(Err::kValue, "mlxturbo_b200 ops take CUDA tensors (there is no CPU path)");
        if (first && t->device() != first->device()) fail(Err::kValue, "%s: tensors must be on one device", what);
        first = first ? first : t;
    }
}

// Packed words [.., K * bits / 32] with scales [.., K / 32]: K.
int64_t mx_check_words(const char* what, const char* name, const at::Tensor& w, const at::Tensor& s, int64_t bits) {
    if (w.element_size() != 4 || w.is_floating_point() || w.dim() < 1)
        fail(Err::kValue, "%s: %s must hold packed 32-bit words", what, name);
    if (s.scalar_type() != at::kByte) fail(Err::kValue, "%s: the scales of %s must be uint8", what, name);
    const int64_t K = w.size(-1) * 32 / bits, lead = w.dim() - 1;
    if (K % 32 || s.dim() != w.dim() || s.size(-1) != K / 32 ||
        s.sizes().slice(0, lead) != w.sizes().slice(0, lead))
        fail(Err::kValue, "%s: the scales of %s have shape %s for words of shape %s", what, name,
             dims(s.sizes()).c_str(), dims(w.sizes()).c_str());
    return K;
}

at::Tensor mx_scratch(const at::Tensor& like, size_t bytes) {
    if (!bytes) return at::Tensor();
    return empty_like_device({(int64_t)bytes + 256}, at::kByte, like);
}
void* mx_scratch_ptr(const at::Tensor& t) {
    return t.defined() ? reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(t.data_ptr()) + 255) & ~(uintptr_t)255)
                       : nullptr;
}

std::tuple<at::Tensor, at::Tensor> mx_quantize(const at::Tensor& v_in, int64_t bits) {
    mx_same_device("quantize", {&v_in});
    const int dt = mx_dtype_code(v_in.scalar_type());
    if (bits != 4 && bits != 8) fail(Err::kNotImplemented, "quantize: bits=%lld", (long long)bits);
    if (v_in.dim() < 1 || v_in.size(-1) == 0 || v_in.size(-1) % 32)
        fail(Err::kValue, "quantize: shape %s: the last axis must be a positive multiple of 32",
             dims(v_in.sizes()).c_str());
    c10::cuda::CUDAGuard guard(v_in.device());
    const at::Tensor v = contiguous16(v_in);
    const int64_t K = v.size(-1), rows = v.numel() / K;
    std::vector<int64_t> shape(v.sizes().begin(), v.sizes().end());
    shape.back() = K * bits / 32;
    at::Tensor w = empty_like_device(shape, at::kInt, v);
    shape.back() = K / 32;
    at::Tensor s = empty_like_device(shape, at::kByte, v);
    check(qmm_mx_quantize(v.data_ptr(), static_cast<uint32_t*>(w.data_ptr()), static_cast<uint8_t*>(s.data_ptr()),
                          rows, K, (int)bits, dt, at::cuda::getCurrentCUDAStream(v.device().index()).stream()),
          "quantize");
    return {w, s};
}

at::Tensor mx_dequantize(const at::Tensor& w_in, const at::Tensor& s_in, int64_t bits, at::ScalarType dtype) {
    mx_same_device("dequantize", {&w_in, &s_in});
    const int dt = mx_dtype_code(dtype);
    if (bits != 4 && bits != 8) fail(Err::kNotImplemented, "dequantize: bits=%lld", (long long)bits);
    const int64_t K = mx_check_words("dequantize", "w", w_in, s_in, bits);
    c10::cuda::CUDAGuard guard(w_in.device());
    const at::Tensor w = contiguous16(w_in), s = s_in.contiguous();
    std::vector<int64_t> shape(w.sizes().begin(), w.sizes().end());
    shape.back() = K;
    at::Tensor out = empty_like_device(shape, dtype, w);
    if (out.numel() == 0) return out;
    check(qmm_mx_dequantize(static_cast<const uint32_t*>(w.data_ptr()), static_cast<const uint8_t*>(s.data_ptr()),
                            out.data_ptr(), out.numel() / K, K, (int)bits, dt,
                            at::cuda::getCurrentCUDAStream(w.device().index()).stream()),
          "dequantize");
    return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> mx_rms_norm(const at::Tensor& x_in,
                                                           const std::optional<at::Tensor>& res_in,
                                                           const at::Tensor& weight_in, double eps) {
    const bool res = res_in.has_value();
    mx_same_device("rms_norm_quantize", {&x_in, res ? &*res_in : nullptr, &weight_in});
    const int dt = mx_half_code(x_in.scalar_type());
    if (x_in.dim() < 1 || x_in.size(-1) == 0 || x_in.size(-1) % 32)
        fail(Err::kValue, "rms_norm_quantize: shape %s: the last axis must be a positive multiple of 32",
             dims(x_in.sizes()).c_str());
    const int64_t K = x_in.size(-1), rows = x_in.numel() / K;
    if (weight_in.dim() != 1 || weight_in.size(0) != K || weight_in.scalar_type() != x_in.scalar_type())
        fail(Err::kValue, "rms_norm_quantize: weight must have shape (%lld) and x's dtype", (long long)K);
    if (res && (res_in->sizes() != x_in.sizes() || res_in->scalar_type() != x_in.scalar_type()))
        fail(Err::kValue, "rms_norm_quantize: residual must have x's shape %s and dtype", dims(x_in.sizes()).c_str());
    if (!(eps >= 0)) fail(Err::kValue, "rms_norm_quantize: eps must not be negative");
    c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = contiguous16(x_in), weight = contiguous16(weight_in);
    at::Tensor r, h;
    if (res) {
        r = contiguous16(*res_in);
        h = empty_like_device(x.sizes(), x.scalar_type(), x);
    }
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = K / 4;
    at::Tensor xq = empty_like_device(shape, at::kInt, x);
    shape.back() = K / 32;
    at::Tensor xs = empty_like_device(shape, at::kByte, x);
    check(qmm_mx_rms_norm(x.data_ptr(), res ? r.data_ptr() : nullptr, weight.data_ptr(), res ? h.data_ptr() : nullptr,
                          static_cast<uint32_t*>(xq.data_ptr()), static_cast<uint8_t*>(xs.data_ptr()), rows, K,
                          (float)eps, dt, at::cuda::getCurrentCUDAStream(x.device().index()).stream()),
          "rms_norm_quantize");
    return {xq, xs, h};
}

// x: values of dtype, or packed mxfp8 words with x_scales; w [N, K/8] mxfp4.
at::Tensor run_mx_matmul(const at::Tensor& x_in, const std::optional<at::Tensor>& xs_in, const at::Tensor& w_in,
                         const at::Tensor& s_in, at::ScalarType dtype, const at::Tensor* out) {
    const bool mx = xs_in.has_value();
    mx_same_device("mx_matmul", {&x_in, mx ? &*xs_in : nullptr, &w_in, &s_in, out});
    const int dt = mx_half_code(dtype);
    if (w_in.dim() != 2) fail(Err::kValue, "mx_matmul: w must be [N, K/8]");
    const int64_t K = mx_check_words("mx_matmul", "w", w_in, s_in, 4), N = w_in.size(0);
    if (x_in.dim() < 1) fail(Err::kValue, "x must have at least one dimension");
    int64_t Kx = x_in.size(-1);
    if (mx) Kx = mx_check_words("mx_matmul", "x", x_in, *xs_in, 8);
    else if (x_in.scalar_type() != dtype) fail(Err::kValue, "mx_matmul: x must have the output's dtype");
    if (Kx != K || K == 0 || N == 0)
        fail(Err::kValue, "mx_matmul: w shape %s does not match K=%lld", dims(w_in.sizes()).c_str(), (long long)Kx);
    c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = contiguous16(x_in), w = contiguous16(w_in), s = s_in.contiguous();
    const at::Tensor xs = mx ? xs_in->contiguous() : at::Tensor();
    const int64_t M = x.numel() / x.size(-1);
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    at::Tensor y;
    if (out) {
        y = *out;
        if (!(y.is_contiguous() && y.sizes() == at::IntArrayRef(shape) && y.scalar_type() == dtype &&
              reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0))
            fail(Err::kValue, "out must be a contiguous, 16-byte aligned tensor of the result shape %s and dtype",
                 dims(at::IntArrayRef(shape)).c_str());
    } else {
        y = empty_like_device(shape, dtype, x);
    }
    if (M == 0) return y;
    const size_t need = qmm_mx_matmul_workspace_size(M, N, K, dt, mx);
    const at::Tensor ws = mx_scratch(x, need);
    check(qmm_mx_matmul(x.data_ptr(), mx ? static_cast<const uint8_t*>(xs.data_ptr()) : nullptr,
                        static_cast<const uint32_t*>(w.data_ptr()), static_cast<const uint8_t*>(s.data_ptr()),
                        y.data_ptr(), M, N, K, dt, mx_scratch_ptr(ws), need,
                        at::cuda::getCurrentCUDAStream(x.device().index()).stream()),
          "mx_matmul");
    return y;
}

at::Tensor mx_matmul(const at::Tensor& x, const std::optional<at::Tensor>& xs, const at::Tensor& w,
                     const at::Tensor& s, at::ScalarType dtype) {
    return run_mx_matmul(x, xs, w, s, dtype, nullptr);
}

at::Tensor& mx_matmul_out(const at::Tensor& x, const std::optional<at::Tensor>& xs, const at::Tensor& w,
                          const at::Tensor& s, at::Tensor& out) {
    run_mx_matmul(x, xs, w, s, out.scalar_type(), &out);
    return out;
}

// x [x_rows, K] or [x_rows, 1, K] (or mxfp8 words), w [E, N, K/8]; lhs / rhs int32 [rows]; y [rows, (1,) N].
at::Tensor mx_gather(const at::Tensor& x_in, const std::optional<at::Tensor>& xs_in, const at::Tensor& w_in,
                     const at::Tensor& s_in, const std::optional<at::Tensor>& lhs_in, const at::Tensor& rhs_in,
                     at::ScalarType dtype, bool sorted) {
    const bool mx = xs_in.has_value(), lhs = lhs_in.has_value();
    mx_same_device("mx_gather", {&x_in, mx ? &*xs_in : nullptr, &w_in, &s_in, lhs ? &*lhs_in : nullptr, &rhs_in});
    const int dt = mx_half_code(dtype);
    if (w_in.dim() != 3) fail(Err::kValue, "w must be [E, N, K/8]");
    const int64_t K = mx_check_words("mx_gather", "w", w_in, s_in, 4), E = w_in.size(0), N = w_in.size(1);
    const bool one = x_in.dim() == 3 && x_in.size(1) == 1;  // [x_rows, 1, K]: y is [rows, 1, N]
    if (x_in.dim() != 2 && !one) fail(Err::kValue, "mx_gather: x must have shape [rows, K] or [rows, 1, K]");
    int64_t Kx = x_in.size(-1);
    if (mx) Kx = mx_check_words("mx_gather", "x", x_in, *xs_in, 8);
    else if (x_in.scalar_type() != dtype) fail(Err::kValue, "mx_gather: x must have the output's dtype");
    if (Kx != K || K == 0 || N == 0 || E == 0)
        fail(Err::kValue, "mx_gather: w shape %s does not match K=%lld", dims(w_in.sizes()).c_str(), (long long)Kx);
    if (rhs_in.scalar_type() != at::kInt || rhs_in.dim() != 1 ||
        (lhs && (lhs_in->scalar_type() != at::kInt || lhs_in->sizes() != rhs_in.sizes())))
        fail(Err::kValue, "mx_gather: indices must be int32 vectors of one length");
    c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = contiguous16(x_in), w = contiguous16(w_in), s = s_in.contiguous(), rhs = rhs_in.contiguous();
    const at::Tensor xs = mx ? xs_in->contiguous() : at::Tensor(), l = lhs ? lhs_in->contiguous() : at::Tensor();
    const int64_t rows = rhs.size(0);
    at::Tensor y = one ? empty_like_device({rows, 1, N}, dtype, x) : empty_like_device({rows, N}, dtype, x);
    if (rows == 0) return y;
    const size_t need = qmm_mx_gather_workspace_size(rows, E, N, K, dt, mx, sorted);
    const at::Tensor ws = mx_scratch(x, need);
    check(qmm_mx_gather(x.data_ptr(), mx ? static_cast<const uint8_t*>(xs.data_ptr()) : nullptr,
                        static_cast<const uint32_t*>(w.data_ptr()), static_cast<const uint8_t*>(s.data_ptr()),
                        lhs ? static_cast<const int32_t*>(l.data_ptr()) : nullptr,
                        static_cast<const int32_t*>(rhs.data_ptr()), y.data_ptr(), rows, x.size(0), E, N, K, dt,
                        sorted, mx_scratch_ptr(ws), need,
                        at::cuda::getCurrentCUDAStream(x.device().index()).stream()),
          "gather_qmm");
    return y;
}

// All-CPU arguments: the same error as a CPU tensor among CUDA ones.
at::Tensor quantized_matmul_cpu(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t,
                                int64_t) {
    fail(Err::kValue, "mlxturbo_b200 ops take CUDA tensors (there is no CPU path)");
}

at::Tensor& quantized_matmul_out_cpu(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                     int64_t, int64_t, at::Tensor& out) {
    fail(Err::kValue, "mlxturbo_b200 ops take CUDA tensors (there is no CPU path)");
}

}  // namespace

TORCH_LIBRARY(mlxturbo_b200, m) {
    m.def("quantized_matmul(Tensor x, Tensor w, Tensor scales, Tensor biases, int group_size=64, int bits=4) "
          "-> Tensor");
    m.def("quantized_matmul_out(Tensor x, Tensor w, Tensor scales, Tensor biases, int group_size, int bits, "
          "*, Tensor(a!) out) -> Tensor(a!)");
    m.def("mx_quantize(Tensor v, int bits) -> (Tensor, Tensor)");
    m.def("mx_dequantize(Tensor w, Tensor scales, int bits, ScalarType dtype) -> Tensor");
    m.def("mx_rms_norm(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("mx_matmul(Tensor x, Tensor? x_scales, Tensor w, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("mx_matmul_out(Tensor x, Tensor? x_scales, Tensor w, Tensor scales, *, Tensor(a!) out) -> Tensor(a!)");
    m.def("mx_gather(Tensor x, Tensor? x_scales, Tensor w, Tensor scales, Tensor? lhs, Tensor rhs, ScalarType dtype, "
          "bool sorted) -> Tensor");
}

// Per device, not for every dispatch key: autograd and the dispatch modes above
// see the calls.  All-CPU arguments reach the same functions, which refuse them.
void mx_impl(torch::Library& m) {
    m.impl("mx_quantize", &mx_quantize);
    m.impl("mx_dequantize", &mx_dequantize);
    m.impl("mx_rms_norm", &mx_rms_norm);
    m.impl("mx_matmul", &mx_matmul);
    m.impl("mx_matmul_out", &mx_matmul_out);
    m.impl("mx_gather", &mx_gather);
}

TORCH_LIBRARY_IMPL(mlxturbo_b200, CUDA, m) {
    m.impl("quantized_matmul", &quantized_matmul);
    m.impl("quantized_matmul_out", &quantized_matmul_out);
    mx_impl(m);
}

TORCH_LIBRARY_IMPL(mlxturbo_b200, CPU, m) {
    m.impl("quantized_matmul", &quantized_matmul_cpu);
    m.impl("quantized_matmul_out", &quantized_matmul_out_cpu);
    mx_impl(m);
}
