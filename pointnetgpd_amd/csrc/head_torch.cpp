// torch binding of the classification-head operators: the autograd nodes of pointnetgpd_amd/head.py, which checks the
// arguments.  In C++ because small layers are bound by the host: a node's backward pass runs on autograd's own thread, and with
// nodes in Python the two threads hand the interpreter to one another.  One forward and backward pass of the classes' loss
// (256 x 256 -> 3, float32) takes 82 us instead of 130, of a linear layer (1531 x 1001 -> 777, float16) 84 instead of 133.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>

#include "pngpd.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<at::Tensor> Maybe;

struct Failure : std::runtime_error {        // _lib.PngpdError in Python
    int code;
    std::string message;
    Failure(int c, const std::string& m) : std::runtime_error("pngpd error " + std::to_string(c) + ": " + m), code(c), message(m) {}
};
void check(int rc) {
    if (rc != PNGPD_OK) throw Failure(rc, pngpd_last_error());
}

int type_of(const at::Tensor& t) {
    return t.scalar_type() == at::kFloat ? PNGPD_TYPE_F32 : t.scalar_type() == at::kBFloat16 ? PNGPD_TYPE_BF16 : PNGPD_TYPE_F16;
}

// A tensor whose memory is rows of `cols` dense elements, `ld` elements apart: a view where the strides allow it, else a copy.
struct Rows {
    at::Tensor t;
    int64_t ld;
    const void* p() const { return t.const_data_ptr(); }
    // rows at 16-byte addresses, whole 16-byte chunks and at most 2^23 bytes apart
    bool aligned() const {
        const int64_t bytes = ld * (int64_t)t.element_size();
        return ((uintptr_t)p() & 15) == 0 && bytes % 16 == 0 && bytes <= (1 << 23);
    }
};
Rows rows_of(const at::Tensor& t, int64_t cols) {
    if (t.is_contiguous()) return {t, cols};
    at::Tensor r = t.reshape({-1, cols});
    if (cols == 1 || r.stride(1) == 1) {
        if (r.size(0) <= 1) return {r, cols};
        if (r.stride(0) >= cols) return {r, r.stride(0)};
    }
    return {r.contiguous(), cols};
}

const void* data(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
at::Tensor dense(const Maybe& t) { return t.has_value() && t->defined() ? t->contiguous() : at::Tensor(); }
bool wants(const at::Tensor& t) { return t.requires_grad(); }
bool wants(const Maybe& t) { return t.has_value() && wants(*t); }

// Forward-mode differentiation: no_grad leaves it on, and a result without its tangent would read as a derivative of zero.
void refuse_tangent(const at::Tensor& t) {
    if (t._fw_grad(0).defined())
        throw std::runtime_error("forward-mode differentiation of this operator is not supported (an input is a dual tensor)");
}
void refuse_tangent(const Maybe& t) {
    if (t.has_value()) refuse_tangent(*t);
}
template <typename... Tensors>
void refuse_tangents(const Tensors&... t) {
    (refuse_tangent(t), ...);
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

// In a capture the engine would make a stream outside it wait for a gradient, or it for the stream, which ends the process.
// That happens where what the gradients go to belongs to such a stream: a leaf whose eager graph is still alive, or an eager
// result.  Called by a backward pass before it launches anything; costs a comparison for each gradient outside a capture.
bool capturing(hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(s, &status) == hipSuccess && status == hipStreamCaptureStatusActive;
}
void refuse_mixed_capture(const at::Tensor& like) {
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const auto current = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.get_device());
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        const auto& edge = node->next_edge(i);
        if (!edge.is_valid() || !node->task_should_compute_output(i)) continue;
        const auto theirs = edge.function->stream();
        if (!theirs.has_value() || *theirs == current.unwrap()) continue;
        if (!capturing(current.stream())) return;
        // the default stream captures nothing, and may not even be asked meanwhile
        const hipStream_t other = c10::hip::HIPStreamMasqueradingAsCUDA(*theirs).stream();
        if (!other || !capturing(other))
            throw std::runtime_error("a captured backward pass reaches a tensor whose eager graph is still alive on another stream: let "
                                     "go of the eager results (a kept loss or output) before the capture");
    }
}

// Gradients are differentiable once: with create_graph each carries a node that raises when it is differentiated.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list defined;
    for (auto& g : grads)
        if (g.defined()) defined.push_back(g.detach().requires_grad_());
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice an operator that is differentiable once", (int)defined.size());
    defined = (*node)(std::move(defined));
    size_t i = 0;
    for (auto& g : grads)
        if (g.defined()) g = defined[i++];
    return grads;
}

// ---- linear ---------------------------------------------------------------------------------------------------------------

at::Tensor linear_forward(const at::Tensor& x, const at::Tensor& w, const Maybe& bias, const Maybe& residual, int64_t act, bool keep,
                          at::Tensor* z) {
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
    const int type = type_of(x);
    const Rows xr = rows_of(x, K), wr = rows_of(w, K);
    Rows rr{at::Tensor(), N};
    if (residual.has_value() && residual->defined()) rr = rows_of(*residual, N);
    const at::Tensor b = dense(bias);
    auto sizes = x.sizes().vec();
    sizes.back() = N;
    at::Tensor y = at::empty(sizes, x.options());
    if (keep && act != PNGPD_ACT_NONE) *z = at::empty({M, N}, x.options());
    const size_t bytes = pngpd_linear_workspace_bytes(type, M, N, K, 0, xr.aligned() && wr.aligned());
    const at::Tensor ws = workspace(bytes, x);
    check(pngpd_linear_forward(type, M, N, K, xr.p(), xr.ld, wr.p(), wr.ld, data(b), (int)act, data(rr.t), rr.ld, out(y), out(*z),
                               out(ws), bytes, stream_of(x)));
    return y;
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const Maybe& bias, const Maybe& residual,
                              int64_t act) {
        at::Tensor z;
        at::Tensor y = linear_forward(x, w, bias, residual, act, wants(x) || wants(w) || wants(bias), &z);
        ctx->save_for_backward({x, w, z});
        ctx->saved_data["args"] = act * 4 + (bias.has_value() ? 1 : 0) + (residual.has_value() ? 2 : 0);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &w = saved[1], &z = saved[2];
        const int64_t args = ctx->saved_data["args"].toInt(), act = args / 4;
        const bool has_b = args & 1, has_r = args & 2;
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const bool need_b = has_b && ctx->needs_input_grad(2), need_r = has_r && ctx->needs_input_grad(2 + (has_b ? 1 : 0));
        variable_list result(5);
        if (!grads[0].defined()) return result;
        refuse_mixed_capture(grads[0]);
        const at::Tensor dy = grads[0].resolve_neg();
        if (need_r) result[3] = dy;
        if (need_x || need_w || need_b) {
            const c10::OptionalDeviceGuard guard(x.device());
            const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
            const int type = type_of(x);
            const Rows xr = rows_of(x, K), wr = rows_of(w, K), dr = rows_of(dy, N);
            if (need_x) result[0] = at::empty(x.sizes(), x.options());
            if (need_w) result[1] = at::empty({N, K}, x.options());
            if (need_b) result[2] = at::empty({N}, x.options());
            const size_t bytes = pngpd_linear_workspace_bytes(type, M, N, K, 1, xr.aligned() && wr.aligned() && dr.aligned());
            const at::Tensor ws = workspace(bytes, x);
            check(pngpd_linear_backward(type, M, N, K, dr.p(), dr.ld, data(z), xr.p(), xr.ld, wr.p(), wr.ld, (int)act, out(result[0]),
                                        out(result[1]), out(result[2]), out(ws), bytes, stream_of(x)));
        }
        return once(std::move(result));
    }
};

at::Tensor linear(const at::Tensor& x, const at::Tensor& w, const Maybe& bias, const Maybe& residual, int64_t act) {
    refuse_tangents(x, w, bias, residual);
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(bias) || wants(residual)))
        return LinearFunction::apply(x, w, bias, residual, act);
    at::Tensor z;
    return linear_forward(x, w, bias, residual, act, false, &z);
}

// ---- dropout --------------------------------------------------------------------------------------------------------------

at::Tensor dropout_call(const at::Tensor& x, const Maybe& residual, double p, uint64_t seed, uint64_t offset, const at::Tensor& rng) {
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t n = x.numel(), cols = x.dim() ? x.size(-1) : 1;
    at::Tensor y = at::empty(x.sizes(), x.options());
    if (n == 0) return y;
    const Rows xr = rows_of(x, cols);
    Rows rr{at::Tensor(), cols};
    if (residual.has_value() && residual->defined()) rr = rows_of(*residual, cols);
    check(pngpd_dropout(type_of(x), n / cols, cols, xr.p(), xr.ld, data(rr.t), rr.ld, out(y), p, seed, offset, (const int64_t*)data(rng),
                        stream_of(x)));
    return y;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const Maybe& residual, double p, int64_t seed, int64_t offset,
                              const Maybe& rng) {
        const at::Tensor r = rng.has_value() ? *rng : at::Tensor();
        ctx->save_for_backward({r});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["residual"] = residual.has_value();
        return dropout_call(x, residual, p, (uint64_t)seed, (uint64_t)offset, r);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        variable_list result(6);
        if (!grads[0].defined()) return result;
        refuse_mixed_capture(grads[0]);
        const at::Tensor dy = grads[0].resolve_neg();
        if (ctx->needs_input_grad(0))
            result[0] = dropout_call(dy, std::nullopt, ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                                     (uint64_t)ctx->saved_data["offset"].toInt(), saved[0]);
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) result[1] = dy;
        return once(std::move(result));
    }
};

at::Tensor dropout(const at::Tensor& x, const Maybe& residual, double p, uint64_t seed, uint64_t offset, const Maybe& rng) {
    refuse_tangents(x, residual);
    if (at::GradMode::is_enabled() && (wants(x) || wants(residual)))
        return DropoutFunction::apply(x, residual, p, (int64_t)seed, (int64_t)offset, rng);
    return dropout_call(x, residual, p, seed, offset, rng.has_value() ? *rng : at::Tensor());
}

// ---- linear + cross entropy -----------------------------------------------------------------------------------------------

struct LossArgs {
    int64_t ignore_index;
    double label_smoothing;
    int64_t reduction;
};

at::Tensor loss_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target, const Maybe& bias, const LossArgs& a,
                        at::Tensor* lse, at::Tensor* kept) {
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t V = w.size(0), D = w.size(1), T = x.numel() / D;
    const int type = type_of(x);
    const Rows xr = rows_of(x, D), wr = rows_of(w, D);
    const at::Tensor b = dense(bias);
    const auto f32 = x.options().dtype(at::kFloat);
    at::Tensor loss = at::empty(a.reduction == PNGPD_REDUCE_NONE ? x.sizes().slice(0, x.dim() - 1) : at::IntArrayRef(), f32);
    *lse = at::empty({T}, f32);
    if (kept) *kept = workspace(pngpd_linear_cross_entropy_kept_bytes(type, T, V, D), x);
    const size_t bytes = pngpd_linear_cross_entropy_workspace_bytes(type, T, V, D, 0, xr.aligned() && wr.aligned());
    const at::Tensor ws = workspace(bytes, x);
    check(pngpd_linear_cross_entropy_forward(type, T, V, D, xr.p(), xr.ld, wr.p(), wr.ld, data(b), target.const_data_ptr<int64_t>(),
                                             a.ignore_index, (float)a.label_smoothing, (int)a.reduction, (float*)out(loss),
                                             (float*)out(*lse), kept ? out(*kept) : nullptr, out(ws), bytes, stream_of(x)));
    return loss;
}

struct LinearCrossEntropyFunction : torch::autograd::Function<LinearCrossEntropyFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const Maybe& bias, const at::Tensor& target,
                              int64_t ignore_index, double label_smoothing, int64_t reduction, bool keep) {
        at::Tensor lse, kept;
        at::Tensor loss = loss_forward(x, w, target, bias, {ignore_index, label_smoothing, reduction}, &lse, keep ? &kept : nullptr);
        ctx->save_for_backward({x, w, dense(bias), target, lse, kept});
        ctx->saved_data["ignore_index"] = ignore_index;
        ctx->saved_data["label_smoothing"] = label_smoothing;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &w = saved[1], &b = saved[2], &target = saved[3], &lse = saved[4];
        variable_list result(8);
        if (!grads[0].defined()) return result;
        refuse_mixed_capture(grads[0]);
        const c10::OptionalDeviceGuard guard(x.device());
        const int64_t V = w.size(0), D = w.size(1), T = x.numel() / D;
        const int type = type_of(x);
        const Rows xr = rows_of(x, D), wr = rows_of(w, D);
        const at::Tensor dloss = grads[0].resolve_neg().contiguous();
        if (ctx->needs_input_grad(0)) result[0] = at::empty(x.sizes(), x.options());
        if (ctx->needs_input_grad(1)) result[1] = at::empty({V, D}, x.options());
        if (b.defined() && ctx->needs_input_grad(2)) result[2] = at::empty({V}, x.options());
        const size_t bytes = pngpd_linear_cross_entropy_workspace_bytes(type, T, V, D, saved[5].defined() ? 2 : 1, xr.aligned() && wr.aligned());
        const at::Tensor ws = workspace(bytes, x);
        check(pngpd_linear_cross_entropy_backward(
            type, T, V, D, xr.p(), xr.ld, wr.p(), wr.ld, data(b), target.const_data_ptr<int64_t>(), ctx->saved_data["ignore_index"].toInt(),
            (float)ctx->saved_data["label_smoothing"].toDouble(), (int)ctx->saved_data["reduction"].toInt(), (const float*)data(lse), data(saved[5]),
            (const float*)data(dloss), out(result[0]), out(result[1]), out(result[2]), out(ws), bytes, stream_of(x)));
        return once(std::move(result));
    }
};

at::Tensor linear_cross_entropy(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target, const Maybe& bias,
                                int64_t ignore_index, double label_smoothing, int64_t reduction, bool keep) {
    refuse_tangents(x, w, bias);
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(bias)))
        return LinearCrossEntropyFunction::apply(x, w, bias, target, ignore_index, label_smoothing, reduction, keep);
    at::Tensor lse;
    return loss_forward(x, w, target, bias, {ignore_index, label_smoothing, reduction}, &lse, nullptr);
}

}  // namespace

PYBIND11_MODULE(_head, m) {
    m.doc() = "autograd nodes of pointnetgpd_amd.head";
    m.attr("built_for") = PNGPD_TORCH;      // "built for torch <version>;"
    pybind11::register_local_exception_translator([](std::exception_ptr e) {
        try {
            if (e) std::rethrow_exception(e);
        } catch (const Failure& f) {
            const auto type = pybind11::module_::import("pointnetgpd_amd._lib").attr("PngpdError");
            PyErr_SetObject(type.ptr(), type(f.code, f.message).ptr());
        }
    });
    const auto unlocked = pybind11::call_guard<pybind11::gil_scoped_release>();
    m.def("linear", &linear, unlocked);
    m.def("dropout", &dropout, unlocked);
    m.def("linear_cross_entropy", &linear_cross_entropy, unlocked);
}
