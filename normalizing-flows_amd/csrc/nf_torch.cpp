// Layer normalisation as a node of torch's autograd graph: the small calls of a conditioner are bound by the host, and a node
// in Python costs more than all of its kernels (256 x 64 fp32, forward + backward: 171 us, with this node 66; the forward pass
// alone 16 and 4.5).  The work itself is in libnf_hip.so (include/nf_hip.h), whose entry points the package hands over once it
// has loaded that library.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <cmath>

#include "../../include/nf_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

struct Library {
    decltype(&nf_layer_norm_fwd) fwd = nullptr;
    decltype(&nf_layer_norm_bwd_workspace_bytes) workspace_bytes = nullptr;
    decltype(&nf_layer_norm_bwd) bwd = nullptr;
    decltype(&nf_strerror) strerror = nullptr;
} lib;

void bind(uintptr_t fwd, uintptr_t workspace_bytes, uintptr_t bwd, uintptr_t strerror) {
    lib.fwd = reinterpret_cast<decltype(lib.fwd)>(fwd);
    lib.workspace_bytes = reinterpret_cast<decltype(lib.workspace_bytes)>(workspace_bytes);
    lib.bwd = reinterpret_cast<decltype(lib.bwd)>(bwd);
    lib.strerror = reinterpret_cast<decltype(lib.strerror)>(strerror);
}

void check(int code, const char* where) {
    TORCH_CHECK(code == 0, where, " failed: ", lib.strerror(code), " (code ", code, ")");
}

int elem_of(at::ScalarType t) { return t == at::kFloat ? NF_ELEM_F32 : t == at::kBFloat16 ? NF_ELEM_BF16 : NF_ELEM_F16; }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// rows as the entry points take them: the tensor itself, or a copy where its last axis is not contiguous (an expanded
// gradient, a transposed view)
Tensor unit_rows(const Tensor& t) {
    return t.size(1) == 1 || t.stride(1) == 1 || !t.numel() ? t : t.contiguous();
}

int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

float* floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

// y, and mean / rstd as the rows of `stats` where it is wanted
Tensor normalise(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0), n = x.size(1);
    Tensor y = at::empty({rows, n}, x.options());
    float* mean = nullptr;
    if (stats) {
        *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
        mean = floats(*stats);
    }
    check(lib.fwd(x.data_ptr(), row_stride(x), floats(weight), floats(bias), y.data_ptr(), n, mean, mean ? mean + rows : nullptr,
                  rows, static_cast<int>(n), eps, elem_of(x.scalar_type()), stream_of(x)),
          "nf_layer_norm_fwd");
    return y;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                          const std::optional<Tensor>& bias, double eps) {
        const Tensor w = weight.value_or(Tensor());
        Tensor stats, y = normalise(x, w, bias.value_or(Tensor()), eps, &stats);
        ctx->save_for_backward({x, w, stats});
        ctx->saved_data["bias"] = bias.has_value();
        return y;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm is differentiable once: create_graph is not supported");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        // (the graph counts the tensors that are there)
        const bool has_w = weight.defined(), has_b = ctx->saved_data["bias"].toBool();
        const bool want_x = ctx->needs_input_grad(0), want_w = has_w && ctx->needs_input_grad(1);
        const bool want_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
        tensor_list out(4);
        if (!grads[0].defined()) return out;
        const c10::DeviceGuard guard(x.device());
        const Tensor g = unit_rows(grads[0]);
        const int64_t rows = x.size(0), n = x.size(1);
        const int elem = elem_of(x.scalar_type());
        const auto single = x.options().dtype(at::kFloat);
        if (want_x) out[0] = at::empty({rows, n}, x.options());
        if (want_w) out[1] = at::empty({n}, single);
        if (want_b) out[2] = at::empty({n}, single);
        const size_t bytes = want_w || want_b ? lib.workspace_bytes(rows, static_cast<int>(n), elem) : 0;
        Tensor workspace;
        if (bytes) workspace = at::empty({static_cast<int64_t>(bytes / sizeof(float))}, single);
        float* mean = floats(stats);
        check(lib.bwd(g.data_ptr(), row_stride(g), x.data_ptr(), row_stride(x), mean, mean + rows, floats(weight),
                      want_x ? out[0].data_ptr() : nullptr, n, floats(out[1]), floats(out[2]), floats(workspace), bytes, rows,
                      static_cast<int>(n), elem, stream_of(x)),
              "nf_layer_norm_bwd");
        return out;
    }
};

std::optional<Tensor> vector(const std::optional<Tensor>& t, const char* name, const Tensor& x) {
    if (!t) return std::nullopt;
    TORCH_CHECK(t->is_cuda(), name, " must be a tensor on the GPU (MI355X); this package has no CPU path");
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, name, " must be float32, got ", t->scalar_type());
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1) && t->device() == x.device(), name, " must be a vector of ",
                      x.size(-1), " elements on ", x.device(), ", got shape ", t->sizes(), " on ", t->device());
    return t->contiguous();
}

// (a tangent of forward-mode differentiation would be dropped without a word)
void check_tangent(const Tensor& t, const char* name) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "layer_norm has no forward-mode derivative: ", name, " carries a tangent");
}

// A leaf whose gradient an earlier graph, still alive, accumulates on the default stream: a backward pass captured with it would
// make that stream wait for the captured one, which no capture allows and which ends the process.  Refused here, before anything
// is recorded.  (Any other stream joins the capture and is joined again at the pass's end: a warm-up on a side stream may keep its
// outputs, hooks may hold an accumulator made there.)
void check_capture(const Tensor& t, const char* name) {
    if (!t.is_leaf() || !t.requires_grad()) return;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!accumulator) return;
    const auto stream = accumulator->stream();
    TORCH_CHECK(!stream || *stream != c10::Stream(c10::Stream::DEFAULT, t.device()), name,
                " takes part in an autograd graph that was recorded on the default stream and is still alive (or a hook holds its "
                "gradient accumulator): before capturing a training step, delete that graph's outputs, or record it and make the "
                "hooks under torch.cuda.stream(a side stream)");
}

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
    TORCH_CHECK(lib.fwd, "libnf_hip.so is not loaded");
    TORCH_CHECK(x.is_cuda(), "x must be a tensor on the GPU (MI355X); this package has no CPU path");
    const auto type = x.scalar_type();
    TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf,
                     "x must be float32, bfloat16 or float16, got ", type);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= INT32_MAX,
                      "x must have a last axis of at least one element, got shape ", x.sizes());
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps must be a finite number >= 0, got ", eps);
    const auto w = vector(weight, "weight", x), b = vector(bias, "bias", x);
    check_tangent(x, "x");
    if (w) check_tangent(*w, "weight");
    if (b) check_tangent(*b, "bias");
    const Tensor rows = unit_rows(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}));
    const bool records = at::GradMode::is_enabled() && (x.requires_grad() || (w && w->requires_grad()) ||
                                                        (b && b->requires_grad()));
    if (records) {
        const c10::DeviceGuard guard(x.device());
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) {
            check_capture(x, "x");
            if (w) check_capture(*weight, "weight");
            if (b) check_capture(*bias, "bias");
        }
    }
    const Tensor y = records ? LayerNormNode::apply(rows, w, b, eps)
                             : normalise(rows, w.value_or(Tensor()), b.value_or(Tensor()), eps, nullptr);
    return x.dim() == 2 ? y : y.view(x.sizes());
}

}  // namespace

PYBIND11_MODULE(_nf_torch, m) {
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"),
          py::call_guard<py::gil_scoped_release>());
}
