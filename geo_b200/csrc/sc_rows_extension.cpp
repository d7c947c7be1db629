// Torch front end of the row operators on 8-bit integers and of the distillation loss: checks of arguments, allocation
// of outputs, current stream and device, autograd.  The kernels are behind the C ABI (include/geo_sc.h).  In C++ and not
// through ctypes like the SC layers' entry points, because the smallest calls (one token, a batch of a few classes) run
// for two microseconds on the device: what a call costs is what the host spends on it.
//
// Arguments are checked before the device is looked at, so that a wrong shape is named on a machine without a GPU too.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <atomic>
#include <optional>
#include <sstream>

#include "geo_sc.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

std::atomic<long long> g_launches{0};   // kernels enqueued through this module

template <typename... A> std::string text(const A &...a) {
    std::ostringstream s;
    (void)std::initializer_list<int>{(s << a, 0)...};
    return s.str();
}
#define REFUSE_TYPE(...) throw py::type_error(text(__VA_ARGS__))
#define REFUSE_VALUE(...) throw py::value_error(text(__VA_ARGS__))

int dtype_code(at::ScalarType t, const char *what) {
    switch (t) {
    case at::kFloat: return GEO_SC_DTYPE_F32;
    case at::kBFloat16: return GEO_SC_DTYPE_BF16;
    case at::kHalf: return GEO_SC_DTYPE_F16;
    default: REFUSE_TYPE(what, " must be float32, bfloat16 or float16, got ", c10::toString(t));
    }
}

void check(int status, const char *what) {
    if (status != GEO_SC_OK) {
        const char *detail = geo_sc_last_error();
        TORCH_CHECK(false, what, ": status ", status, " (", *detail ? detail : geo_sc_status_string(status), ")");
    }
}

void check_rows(const Tensor &t, const char *what) {
    if (t.dim() < 1 || t.size(-1) < 1) REFUSE_VALUE(what, " needs a last dimension of at least 1, got shape ", t.sizes());
    if (t.size(-1) > INT32_MAX || t.numel() / t.size(-1) > INT32_MAX)
        REFUSE_VALUE(what, " has more than 2^31 - 1 rows or columns: ", t.sizes());
}

void one_device(std::initializer_list<const Tensor *> tensors) {
    const Tensor *first = nullptr;
    for (const Tensor *t : tensors) {
        if (!t) continue;
        TORCH_CHECK(t->is_cuda(), "geo_b200 kernels run on CUDA tensors only (there is no CPU path)");
        if (!first) first = t;
        else if (t->device() != first->device()) REFUSE_VALUE("tensors on ", first->device(), " and ", t->device(), " in one call");
    }
}

void evaluation_only(const char *name, std::initializer_list<const Tensor *> tensors) {
    // a gradient is asked for under grad mode only, a tangent (forward mode) whatever that is
    const bool grad = at::GradMode::is_enabled(), tangent = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Tensor *t : tensors) {
        if (!t) continue;
        TORCH_CHECK(!grad || !t->requires_grad(), name, " has no gradient (evaluation only): call it under torch.no_grad() or detach its inputs");
        TORCH_CHECK(!tangent || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative (evaluation only): give it the primal values");
    }
}

const Tensor *ptr(const OptTensor &t) { return t.has_value() && t->defined() ? &*t : nullptr; }
void *data(const Tensor *t) { return t ? t->data_ptr() : nullptr; }

// `t` as [rows, last dimension] with dense rows: a view where the strides allow one.
Tensor rows_of(const Tensor &t) {
    const Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)});
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

// Uninitialised output on the device, past the dispatcher (a third of what an allocation costs the host).
Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, at::Device device) {
    return at::detail::empty_cuda(sizes, dtype, device, std::nullopt);
}

// int8 [rows, cols] whose rows start on 16-byte boundaries, as the product reads them.
Tensor empty_rows(int64_t rows, int64_t cols, at::Device device) {
    const int64_t padded = (cols + 15) / 16 * 16;
    const Tensor t = new_tensor({rows, padded}, at::kChar, device);
    return padded == cols ? t : t.narrow(1, 0, cols);
}

Tensor aligned_rows(const Tensor &t) {
    if (t.stride(1) == 1 && t.stride(0) % 16 == 0 && t.stride(0) >= t.size(1) && (uintptr_t)t.data_ptr() % 16 == 0) return t;
    return empty_rows(t.size(0), t.size(1), t.device()).copy_(t);
}

Tensor like_rows(const Tensor &q, const Tensor &x) {   // [rows, cols] back to the leading dimensions of x
    return x.dim() == 2 ? q : x.dim() == 1 ? q.select(0, 0) : q.unflatten(0, x.sizes().slice(0, x.dim() - 1));
}

py::tuple rms_norm_int8(const Tensor &x, const Tensor &weight, const OptTensor &residual_, double eps) {
    const Tensor *residual = ptr(residual_);
    const int code = dtype_code(x.scalar_type(), "x");
    dtype_code(weight.scalar_type(), "weight");
    check_rows(x, "x");
    const int64_t cols = x.size(-1);
    if (weight.dim() != 1 || weight.size(0) != cols) REFUSE_VALUE("weight has shape ", weight.sizes(), ", expected [", cols, "]");
    if (residual && (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type()))
        REFUSE_VALUE("residual is ", residual->scalar_type(), residual->sizes(), ", x is ", x.scalar_type(), x.sizes());
    if (!(eps >= 0.0 && eps < 3.4e38)) REFUSE_VALUE("eps must be finite and not negative, got ", eps);
    evaluation_only("rms_norm_int8", {&x, &weight, residual});
    one_device({&x, &weight, residual});
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x.device());
    // the kernels take the weight in fp32 or in the type of x
    const Tensor xr = rows_of(x), w = (weight.scalar_type() == x.scalar_type() ? weight : weight.to(at::kFloat)).contiguous();
    const int wcode = dtype_code(w.scalar_type(), "weight");
    const int64_t rows = xr.size(0);
    const Tensor q = empty_rows(rows, cols, x.device()), scale = new_tensor(x.sizes().slice(0, x.dim() - 1), at::kFloat, x.device());
    Tensor rr, total;
    if (residual) {
        rr = rows_of(*residual);
        total = new_tensor(x.sizes(), x.scalar_type(), x.device());
    }
    check(geo_sc_rms_norm_int8(rows, (int)cols, code, xr.data_ptr(), xr.stride(0), residual ? rr.data_ptr() : nullptr,
                               residual ? rr.stride(0) : 0, w.data_ptr(), wcode, (float)eps, residual ? total.data_ptr() : nullptr,
                               (int8_t *)q.data_ptr(), q.stride(0), (float *)scale.data_ptr(), c10::cuda::getCurrentCUDAStream().stream()),
          "geo_sc_rms_norm_int8");
    g_launches += rows > 0;
    return residual ? py::make_tuple(like_rows(q, x), scale, total) : py::make_tuple(like_rows(q, x), scale);
}

py::tuple quantize_int8(const Tensor &x) {
    const int code = dtype_code(x.scalar_type(), "x");
    check_rows(x, "x");
    evaluation_only("quantize_int8", {&x});
    one_device({&x});
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor xr = rows_of(x);
    const Tensor q = empty_rows(xr.size(0), xr.size(1), x.device()), scale = new_tensor(x.sizes().slice(0, x.dim() - 1), at::kFloat, x.device());
    check(geo_sc_quantize_int8(xr.size(0), (int)xr.size(1), code, xr.data_ptr(), xr.stride(0), (int8_t *)q.data_ptr(), q.stride(0),
                               (float *)scale.data_ptr(), c10::cuda::getCurrentCUDAStream().stream()),
          "geo_sc_quantize_int8");
    g_launches += xr.size(0) > 0;
    return py::make_tuple(like_rows(q, x), scale);
}

Tensor dequantize_int8(const Tensor &q, const Tensor &scale, at::ScalarType dtype) {
    const int code = dtype_code(dtype, "dtype");
    if (q.scalar_type() != at::kChar || scale.scalar_type() != at::kFloat)
        REFUSE_TYPE("q must be int8 and scale float32, got ", q.scalar_type(), " and ", scale.scalar_type());
    check_rows(q, "q");
    if (scale.sizes() != q.sizes().slice(0, q.dim() - 1)) REFUSE_VALUE("scale has shape ", scale.sizes(), ", q ", q.sizes());
    evaluation_only("dequantize_int8", {&scale});
    one_device({&q, &scale});
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(q.device());
    const Tensor qr = rows_of(q), s = scale.contiguous(), out = new_tensor(q.sizes(), dtype, q.device());
    check(geo_sc_dequantize_int8(qr.size(0), (int)qr.size(1), (const int8_t *)qr.data_ptr(), qr.stride(0), (const float *)s.data_ptr(), code,
                                 out.data_ptr(), c10::cuda::getCurrentCUDAStream().stream()),
          "geo_sc_dequantize_int8");
    g_launches += qr.size(0) > 0;
    return out;
}

Tensor linear_int8(const Tensor &q, const Tensor &scale, const Tensor &weight_q, const Tensor &weight_scale, const OptTensor &bias_,
                   at::ScalarType dtype) {
    const Tensor *bias = ptr(bias_);
    const int code = dtype_code(dtype, "dtype");
    if (q.scalar_type() != at::kChar || weight_q.scalar_type() != at::kChar)
        REFUSE_TYPE("the operands must be int8, got ", q.scalar_type(), " and ", weight_q.scalar_type());
    if (scale.scalar_type() != at::kFloat || weight_scale.scalar_type() != at::kFloat || (bias && bias->scalar_type() != at::kFloat))
        REFUSE_TYPE("scales and bias must be float32");
    check_rows(q, "q");
    if (weight_q.dim() != 2 || weight_q.size(0) < 1 || weight_q.size(1) != q.size(-1))
        REFUSE_VALUE("feature mismatch: q is ", q.sizes(), ", weight ", weight_q.sizes());
    check_rows(weight_q, "weight");
    const int64_t n = weight_q.size(0), k = weight_q.size(1);
    if (scale.sizes() != q.sizes().slice(0, q.dim() - 1) || weight_scale.dim() != 1 || weight_scale.size(0) != n ||
        (bias && (bias->dim() != 1 || bias->size(0) != n)))
        REFUSE_VALUE("scales ", scale.sizes(), " and ", weight_scale.sizes(), " or the bias do not match the rows of ", q.sizes(), " and ",
                     weight_q.sizes());
    if (k > 131071) REFUSE_VALUE("k = ", k, ": sums of more than 131071 products may leave 32 bits");
    evaluation_only("linear_int8", {&scale, &weight_scale, bias});
    one_device({&q, &scale, &weight_q, &weight_scale, bias});
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(q.device());
    const Tensor x = aligned_rows(rows_of(q)), w = aligned_rows(weight_q);
    const Tensor s = scale.contiguous(), ws = weight_scale.contiguous();
    Tensor b;
    if (bias) b = bias->contiguous();
    const int64_t m = x.size(0);
    at::DimVector shape(q.sizes());
    shape.back() = n;
    const Tensor out = new_tensor(shape, dtype, q.device());
    check(geo_sc_linear_int8((int)m, (int)n, (int)k, (const int8_t *)x.data_ptr(), x.stride(0), (const float *)s.data_ptr(),
                             (const int8_t *)w.data_ptr(), w.stride(0), (const float *)ws.data_ptr(), bias ? (const float *)b.data_ptr() : nullptr,
                             code, out.data_ptr(), n, c10::cuda::getCurrentCUDAStream().stream()),
          "geo_sc_linear_int8");
    g_launches += m > 0;
    return out;
}

// The graph capture that the current stream is part of; 0: none.
int64_t capture_id() {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    C10_CUDA_CHECK(cudaStreamGetCaptureInfo(c10::cuda::getCurrentCUDAStream().stream(), &status, &id));
    return status == cudaStreamCaptureStatusActive ? (int64_t)id : 0;
}

// The loss with its gradient.  With a scalar loss the forward pass writes the gradient for an upstream gradient of 1
// along with the loss, so that the logits are read once; the backward pass hands that over, writing it anew (decided on
// the device) where the upstream gradient is another.  A second backward pass over the same graph writes its own, and so
// does one on the other side of a graph capture: replayed without the forward pass, it would find what an earlier replay
// or the gradient's owner has left in that memory.
struct Distillation : torch::autograd::Function<Distillation> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &logits, const Tensor &indices, const Tensor &teacher,
                          const OptTensor &weight_, double temperature, double scale, bool mean, bool need) {
        const Tensor weight = weight_.value_or(Tensor());
        c10::cuda::CUDAGuard guard(logits.device());
        const Tensor z = rows_of(logits);
        const int64_t rows = z.size(0), vocab = z.size(1);
        const Tensor row_loss = new_tensor(logits.sizes().slice(0, logits.dim() - 1), at::kFloat, logits.device());
        const Tensor stats = new_tensor({rows, 2}, at::kFloat, logits.device());
        Tensor loss, grad;
        if (mean) loss = new_tensor({}, at::kFloat, logits.device());
        if (mean && need) grad = new_tensor(logits.sizes(), logits.scalar_type(), logits.device());
        check(geo_sc_distill_forward(rows, (int)vocab, (int)indices.size(-1), dtype_code(logits.scalar_type(), "logits"), z.data_ptr(),
                                     z.stride(0), indices.data_ptr(), indices.scalar_type() == at::kLong ? 64 : 32, teacher.data_ptr(),
                                     dtype_code(teacher.scalar_type(), "teacher_logits"),
                                     weight.defined() ? (const float *)weight.data_ptr() : nullptr, (float)temperature, (float)scale, mean,
                                     (float *)row_loss.data_ptr(), stats.data_ptr(), mean ? (float *)loss.data_ptr() : nullptr,
                                     grad.defined() ? grad.data_ptr() : nullptr, c10::cuda::getCurrentCUDAStream().stream()),
              "geo_sc_distill_forward");
        g_launches += (rows > 0) + mean;
        if (need) {
            ctx->save_for_backward({logits, indices, teacher, weight, stats});
            ctx->saved_data["temperature"] = temperature;
            ctx->saved_data["scale"] = scale;
            ctx->saved_data["mean"] = mean;
            if (grad.defined()) {
                ctx->saved_data["ready"] = grad;
                ctx->saved_data["capture"] = capture_id();
            }
        }
        return mean ? loss : row_loss;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list upstream) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &indices = saved[1], &teacher = saved[2], &weight = saved[3], &stats = saved[4];
        const bool mean = ctx->saved_data["mean"].toBool(), again = at::GradMode::is_enabled();
        Tensor grad;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(logits.device());
            const Tensor z = rows_of(logits), up = upstream[0].to(at::kFloat).contiguous();
            bool ready = false;
            const auto it = ctx->saved_data.find("ready");
            if (it != ctx->saved_data.end() && ctx->saved_data["capture"].toInt() == capture_id()) {
                grad = it->second.toTensor();
                ctx->saved_data.erase(it);
                ready = true;
            } else {
                grad = new_tensor(logits.sizes(), logits.scalar_type(), logits.device());
            }
            check(geo_sc_distill_backward(z.size(0), (int)z.size(1), (int)indices.size(-1), dtype_code(logits.scalar_type(), "logits"),
                                          z.data_ptr(), z.stride(0), indices.data_ptr(), indices.scalar_type() == at::kLong ? 64 : 32,
                                          teacher.data_ptr(), dtype_code(teacher.scalar_type(), "teacher_logits"),
                                          weight.defined() ? (const float *)weight.data_ptr() : nullptr,
                                          (float)ctx->saved_data["temperature"].toDouble(), (float)ctx->saved_data["scale"].toDouble(), mean,
                                          stats.data_ptr(), (const float *)up.data_ptr(), ready, grad.data_ptr(),
                                          c10::cuda::getCurrentCUDAStream().stream()),
                  "geo_sc_distill_backward");
            g_launches += z.size(0) > 0;
        }
        if (again) {   // create_graph: the gradient itself has none
            auto error = std::make_shared<torch::autograd::DelayedError>("distillation_loss can be differentiated only once", 1);
            Tensor leaf = grad.detach();
            leaf.requires_grad_(true);
            grad = (*error)({leaf})[0];
        }
        return {grad, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor distillation_loss(const Tensor &logits, const Tensor &indices, const Tensor &teacher, double temperature, const OptTensor &weight_,
                         const std::string &reduction, double scale) {
    const Tensor *weight = ptr(weight_);
    dtype_code(logits.scalar_type(), "logits");
    dtype_code(teacher.scalar_type(), "teacher_logits");
    if (reduction != "batchmean" && reduction != "sum" && reduction != "none")
        REFUSE_VALUE("reduction must be 'batchmean', 'sum' or 'none', got '", reduction, "'");
    if (indices.scalar_type() != at::kLong && indices.scalar_type() != at::kInt)
        REFUSE_TYPE("indices must be int64 or int32, got ", indices.scalar_type());
    check_rows(logits, "logits");
    const auto rows = logits.sizes().slice(0, logits.dim() - 1);
    if (indices.dim() != logits.dim() || indices.sizes() != teacher.sizes() || indices.sizes().slice(0, indices.dim() - 1) != rows)
        REFUSE_VALUE("logits ", logits.sizes(), ", indices ", indices.sizes(), " and teacher_logits ", teacher.sizes(), " do not match");
    if (indices.size(-1) < 1 || indices.size(-1) > 512) REFUSE_VALUE("between 1 and 512 entries per row, got ", indices.size(-1));
    if (weight && (weight->sizes() != rows || weight->scalar_type() != at::kFloat))
        REFUSE_VALUE("weight must be float32 of shape ", rows, ", got ", weight->scalar_type(), weight->sizes());
    if (!(temperature >= 1e-6 && temperature <= 1e6)) REFUSE_VALUE("temperature must lie in [1e-6, 1e6], got ", temperature);
    if (reduction == "sum") scale *= std::max<int64_t>(1, logits.numel() / logits.size(-1));   // the kernels divide by the rows
    if (!(std::abs(scale) < 3.4e38)) REFUSE_VALUE("scale (for a sum, times the number of rows) must be finite in 32 bits, got ", scale);
    const bool grad_mode = at::GradMode::is_enabled();
    if (grad_mode && (teacher.requires_grad() || (weight && weight->requires_grad())))
        REFUSE_VALUE("distillation_loss has no gradient for teacher_logits and weight: detach them");
    one_device({&logits, &indices, &teacher, weight});
    return Distillation::apply(logits, indices.contiguous(), teacher.contiguous(), weight ? OptTensor(weight->contiguous()) : OptTensor(), temperature, scale,
                               reduction != "none", grad_mode && logits.requires_grad());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("rms_norm_int8", &rms_norm_int8);
    m.def("quantize_int8", &quantize_int8);
    m.def("dequantize_int8", [](const Tensor &q, const Tensor &scale, const py::object &dtype) {
        return dequantize_int8(q, scale, torch::python::detail::py_object_to_dtype(dtype));
    });
    m.def("linear_int8", [](const Tensor &q, const Tensor &scale, const Tensor &wq, const Tensor &ws, const OptTensor &bias, const py::object &dtype) {
        return linear_int8(q, scale, wq, ws, bias, torch::python::detail::py_object_to_dtype(dtype));
    });
    m.def("distillation_loss", &distillation_loss);
    m.def("launches", []() { return g_launches.load(); });
}
