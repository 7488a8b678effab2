// The training-side operators as torch functions: argument checks, output and scratch tensors, the current
// stream and the autograd nodes, on top of the C ABI (include/scmiac_hip.h).
//
// These run once or more per training step of a few hundred microseconds, where a Python autograd function and a
// ctypes call cost more than the kernels.  The library is bound by path at import (bind), so that this module and
// the ctypes binding use the same one.
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/scmiac_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------ the library

struct Library {
    decltype(&scmiac_last_error) last_error = nullptr;
    decltype(&scmiac_linear_workspace_size) linear_workspace_size;
    decltype(&scmiac_linear_forward) linear_forward;
    decltype(&scmiac_linear_backward) linear_backward;
    decltype(&scmiac_top_logits_workspace_size) top_logits_workspace_size;
    decltype(&scmiac_top_logits) top_logits;
    decltype(&scmiac_distill_workspace_size) distill_workspace_size;
    decltype(&scmiac_distill_forward) distill_forward;
    decltype(&scmiac_distill_backward) distill_backward;
} lib;

void bind(const std::string& path) {
    void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(handle, "cannot load ", path, ": ", dlerror());
    Library l;
    auto get = [&](auto& fn, const char* name) {
        void* at = dlsym(handle, name);
        TORCH_CHECK(at, path, " has no ", name);
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at);
    };
    get(l.linear_workspace_size, "scmiac_linear_workspace_size");
    get(l.linear_forward, "scmiac_linear_forward");
    get(l.linear_backward, "scmiac_linear_backward");
    get(l.top_logits_workspace_size, "scmiac_top_logits_workspace_size");
    get(l.top_logits, "scmiac_top_logits");
    get(l.distill_workspace_size, "scmiac_distill_workspace_size");
    get(l.distill_forward, "scmiac_distill_forward");
    get(l.distill_backward, "scmiac_distill_backward");
    get(l.last_error, "scmiac_last_error");
    lib = l;
}

// ValueError for bad arguments, RuntimeError for the rest
void check(int rc) {
    if (rc == SCMIAC_OK) return;
    const char* why = lib.last_error();
    TORCH_CHECK_VALUE(rc != SCMIAC_ERR_ARG, "libscmiac_hip status ", rc, ": ", why);
    TORCH_CHECK(false, "libscmiac_hip status ", rc, ": ", why);
}

// ------------------------------------------------------------------ tensors

int dtype_code(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return SCMIAC_F32;
        case at::kHalf: return SCMIAC_F16;
        case at::kBFloat16: return SCMIAC_BF16;
        default: TORCH_CHECK_TYPE(false, what, " must be float32, float16 or bfloat16, not ", t.scalar_type());
    }
}

// The kernels read memory as it is: a negation that a view has pending (imag of a conjugate) is carried out first.
Tensor as_stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// The kernels take device pointers: a host pointer handed to them is a memory fault, not an exception.
Tensor on_gpu(const OptTensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.has_value() && t->defined() && t->is_cuda(), what, " must be a tensor on a GPU device (got ",
                      t.has_value() && t->defined() ? t->device().str() : std::string("none"), "); there is no CPU path");
    return as_stored(*t);
}
Tensor on_gpu(const OptTensor& t, const char* what, const Tensor& beside) {
    const Tensor v = on_gpu(t, what);
    TORCH_CHECK_VALUE(v.device() == beside.device(), what, " is on ", v.device(), ", not on ", beside.device());
    return v;
}

// A recorder of torch's operators would see the outputs made and never what fills them.
void no_recorder() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                "this operator cannot be traced (torch.jit.trace, torch.export, make_fx)");
}

// An input with a tangent (torch.autograd.forward_ad) would lose it.
void no_tangent(const OptTensor& t, const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t), what, " has a tangent: this operator has no forward-mode derivative");
}

// a 2-D tensor whose columns lie next to each other, and its row stride
struct Rows {
    Tensor t;
    int64_t ld = 0;
    Rows() = default;
    explicit Rows(const Tensor& v) {
        if (!v.defined()) return;
        t = v.size(1) == 1 || v.stride(1) == 1 ? v : v.contiguous();
        ld = t.stride(0);
    }
    const void* data() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void* in_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// Scratch of one call: it belongs to the stream, or to the graph under capture, that the call runs on, so that
// calls on two streams and two captured graphs never share it.
struct Scratch {
    Tensor t;
    size_t bytes = 0;
    void* data() const { return out_ptr(t); }
    void make(const Tensor& beside) {
        if (bytes) t = at::empty({static_cast<int64_t>(bytes)}, beside.options().dtype(at::kByte));
    }
};
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Gradients of a backward pass that was itself recorded (create_graph) have no derivative: a node that says so stands
// between them and every input of the pass that requires a gradient, whether or not it was kept for this pass, and
// the gradient `given` to it.
void close(variable_list& grads, const Tensor& given) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list edges;
    const std::shared_ptr<torch::autograd::Node> self = torch::autograd::get_current_node();
    TORCH_CHECK(self, "create_graph needs the autograd engine");
    for (const torch::autograd::Edge& e : self->next_edges())
        if (e.is_valid()) edges.push_back(e);
    if (given.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(given));
    const std::shared_ptr<torch::autograd::Node> last(
        new torch::autograd::Error("this operator is not differentiable twice", std::move(edges)), torch::autograd::deleteNode);
    for (Tensor& g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::set_history(g, last);
        }
}

// ------------------------------------------------------------------ dense layer

Tensor linear_forward(const Tensor& x_, const Tensor& w_, const Tensor& bias_, const Tensor& residual_, int64_t act, bool keep,
                      Tensor* z) {
    const c10::DeviceGuard guard(x_.device());
    const Rows x(x_), w(w_), residual(residual_);
    const Tensor bias = bias_.defined() ? bias_.contiguous() : bias_;
    const int64_t m = x_.size(0), k = x_.size(1), n = w_.size(0);
    const int code = dtype_code(x_, "x");
    Scratch ws;
    check(lib.linear_workspace_size(m, n, k, code, (int)act, 0, &ws.bytes));
    ws.make(x_);
    Tensor y = at::empty({m, n}, x_.options());
    if (keep && act != SCMIAC_ACT_NONE) *z = at::empty({m, n}, x_.options());
    check(lib.linear_forward(x.data(), x.ld, w.data(), w.ld, in_ptr(bias), residual.data(), residual.ld, m, n, k, code, (int)act,
                             out_ptr(y), z ? out_ptr(*z) : nullptr, ws.data(), ws.bytes, stream_of(x_)));
    return y;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_, const OptTensor& residual_,
                          int64_t act) {
        const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
        const bool need_x = x.requires_grad(), need_w = w.requires_grad(), need_b = bias.defined() && bias.requires_grad();
        Tensor z;
        Tensor y = linear_forward(x, w, bias, residual, act, need_x || need_w || need_b, &z);
        ctx->save_for_backward({need_w ? x : Tensor(), need_x ? w : Tensor(), z});
        ctx->saved_data["act"] = act;
        ctx->saved_data["k"] = x.size(1);
        // the inputs' numbers in needs_input_grad, which counts the tensors there are
        ctx->saved_data["bias"] = bias.defined() ? 2 : -1;
        ctx->saved_data["residual"] = residual.defined() ? 2 + (int64_t)bias.defined() : -1;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        auto needed = [&](int64_t at) { return at >= 0 && ctx->needs_input_grad(at); };
        const bool need_x = needed(0) && saved[1].defined(), need_w = needed(1) && saved[0].defined(),
                   need_b = needed(ctx->saved_data["bias"].toInt());
        const Tensor& given = grads[0];
        variable_list out(5);
        if (need_x || need_w || need_b) {
            const at::NoGradGuard no_grad;
            const c10::DeviceGuard guard(given.device());
            const int64_t act = ctx->saved_data["act"].toInt(), k = ctx->saved_data["k"].toInt();
            const Rows x(need_w ? saved[0] : Tensor()), w(need_x ? saved[1] : Tensor());
            const Tensor dy = as_stored(given).contiguous();
            const int64_t m = dy.size(0), n = dy.size(1);
            const int code = dtype_code(dy, "the gradient");
            Scratch ws;
            check(lib.linear_workspace_size(m, n, k, code, (int)act, 1, &ws.bytes));
            ws.make(dy);
            if (need_x) out[0] = at::empty({m, k}, dy.options());
            if (need_w) out[1] = at::empty({n, k}, dy.options());
            if (need_b) out[2] = at::empty({n}, dy.options());
            check(lib.linear_backward(x.data(), x.ld, w.data(), w.ld, in_ptr(saved[2]), in_ptr(dy), m, n, k, code, (int)act,
                                      out_ptr(out[0]), out_ptr(out[1]), out_ptr(out[2]), ws.data(), ws.bytes, stream_of(dy)));
        }
        close(out, given);
        if (needed(ctx->saved_data["residual"].toInt())) out[3] = given;      // (itself, with whatever derivatives it has)
        return out;
    }
};

OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

Tensor linear_act(const OptTensor& x_, const OptTensor& w_, const OptTensor& bias_, const OptTensor& residual_, int64_t act) {
    no_recorder();
    const Tensor x = on_gpu(x_, "x");
    const Tensor w = on_gpu(w_, "weight", x);
    dtype_code(x, "x");
    const Tensor bias = bias_.has_value() ? on_gpu(bias_, "bias", x) : Tensor();
    const Tensor residual = residual_.has_value() ? on_gpu(residual_, "residual", x) : Tensor();
    no_tangent(x_, "x"), no_tangent(w_, "weight"), no_tangent(bias_, "bias"), no_tangent(residual_, "residual");
    TORCH_CHECK_TYPE(w.scalar_type() == x.scalar_type(), "weight is ", w.scalar_type(), ", x is ", x.scalar_type());
    TORCH_CHECK_TYPE(!bias.defined() || bias.scalar_type() == x.scalar_type(), "bias is ", bias.scalar_type(), ", x is ", x.scalar_type());
    TORCH_CHECK_TYPE(!residual.defined() || residual.scalar_type() == x.scalar_type(), "residual is ", residual.scalar_type(), ", x is ",
                     x.scalar_type());
    TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1) && w.size(0) > 0 && w.size(1) > 0,
                      "x [..., k] and weight [n, k] do not match: ", x.sizes(), ", ", w.sizes());
    const bool flat = x.dim() == 2;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = w.size(0);
    TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == w.size(0)), "bias needs shape [", w.size(0), "], not ",
                      bias.sizes());
    TORCH_CHECK_VALUE(!residual.defined() || residual.sizes() == at::IntArrayRef(shape), "residual needs shape ", at::IntArrayRef(shape),
                      ", not ", residual.sizes());
    const Tensor x2 = flat ? x : x.reshape({-1, x.size(-1)});
    const Tensor r2 = flat || !residual.defined() ? residual : residual.reshape({-1, w.size(0)});
    const bool grads = at::GradMode::is_enabled() &&
                       (x2.requires_grad() || w.requires_grad() || (bias.defined() && bias.requires_grad()) || (r2.defined() && r2.requires_grad()));
    const Tensor y = grads ? LinearAct::apply(x2, w, given(bias), given(r2), act) : linear_forward(x2, w, bias, r2, act, false, nullptr);
    return flat ? y : y.view(shape);
}

// ------------------------------------------------------------------ top logits

std::tuple<Tensor, Tensor, Tensor> top_logits(const OptTensor& logits_, int64_t k, double temperature) {
    no_recorder();
    const Tensor logits = on_gpu(logits_, "logits").detach();
    const int code = dtype_code(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits need at least one class");
    TORCH_CHECK_VALUE(k >= 1 && k <= SCMIAC_TOP_MAX_K, "k=", k, " outside 1..", SCMIAC_TOP_MAX_K);
    const c10::DeviceGuard guard(logits.device());
    const bool flat = logits.dim() == 2;
    const Rows x(flat ? logits : logits.reshape({-1, logits.size(-1)}));
    const int64_t n = x.t.size(0), v = x.t.size(1);
    Scratch ws;
    check(lib.top_logits_workspace_size(n, v, (int)k, code, &ws.bytes));
    ws.make(logits);
    Tensor values = at::empty({n, k}, logits.options()), idx = at::empty({n, k}, logits.options().dtype(at::kInt)),
           lse = at::empty({n}, logits.options().dtype(at::kFloat));
    check(lib.top_logits(x.data(), x.ld, n, v, code, (int)k, (float)temperature, out_ptr(values), idx.mutable_data_ptr<int32_t>(),
                         lse.mutable_data_ptr<float>(), ws.data(), ws.bytes, stream_of(logits)));
    if (flat) return {values, idx, lse};
    std::vector<int64_t> rows(logits.sizes().begin(), logits.sizes().end() - 1), table = rows;
    table.push_back(k);
    return {values.view(table), idx.view(table), lse.view(rows)};
}

// ------------------------------------------------------------------ distillation

struct Teacher {
    Tensor idx, top, lse;      // int32 [n, k], float32 [n, k], float32 [n] or undefined; contiguous
    double temperature, own_temperature;
};

std::tuple<Tensor, Tensor, Tensor> distill_forward(const Tensor& logits, const Teacher& t, int64_t reduction) {
    const c10::DeviceGuard guard(logits.device());
    const Rows x(logits);
    const int64_t n = x.t.size(0), v = x.t.size(1);
    const int code = dtype_code(logits, "logits");
    const at::TensorOptions f32 = logits.options().dtype(at::kFloat);
    Scratch ws;
    check(lib.distill_workspace_size(n, v, code, &ws.bytes));
    ws.make(logits);
    Tensor stats = at::empty({n, 4}, f32), loss = reduction == SCMIAC_REDUCE_NONE ? at::empty({n}, f32) : at::empty({}, f32), scale;
    if (reduction != SCMIAC_REDUCE_NONE) scale = at::empty({}, f32);
    check(lib.distill_forward(x.data(), x.ld, n, v, code, t.idx.const_data_ptr<int32_t>(), t.top.const_data_ptr<float>(),
                              (int)t.idx.size(1), static_cast<const float*>(in_ptr(t.lse)), (float)t.temperature,
                              (float)t.own_temperature, (int)reduction, loss.mutable_data_ptr<float>(), stats.mutable_data_ptr<float>(),
                              static_cast<float*>(out_ptr(scale)), ws.data(), ws.bytes, stream_of(logits)));
    return {loss, stats, scale};
}

struct TopkDistill : torch::autograd::Function<TopkDistill> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& idx, const Tensor& top, const OptTensor& lse,
                          double temperature, double own_temperature, int64_t reduction) {
        auto [loss, stats, scale] = distill_forward(logits, {idx, top, lse.value_or(Tensor()), temperature, own_temperature}, reduction);
        ctx->save_for_backward({logits, idx, top, stats, scale});
        ctx->saved_data["t"] = temperature;
        ctx->saved_data["ta"] = own_temperature;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &idx = saved[1], &top = saved[2], &stats = saved[3], &scale = saved[4];
        const Tensor grad = as_stored(grads[0]);
        variable_list out(7);
        {
            const at::NoGradGuard no_grad;
            const c10::DeviceGuard guard(logits.device());
            const Rows x(logits);
            const int64_t n = x.t.size(0), v = x.t.size(1);
            // rows as far apart as x's where those are padded: both then start alike with respect to 16 bytes
            const int64_t ldd = x.ld >= v && x.ld <= 2 * v ? x.ld : v;
            Tensor dx = at::empty({n, ldd}, logits.options());
            if (ldd != v) dx = dx.narrow(1, 0, v);
            check(lib.distill_backward(x.data(), x.ld, n, v, dtype_code(logits, "logits"), idx.const_data_ptr<int32_t>(),
                                       top.const_data_ptr<float>(), (int)idx.size(1), (float)ctx->saved_data["t"].toDouble(),
                                       (float)ctx->saved_data["ta"].toDouble(), stats.const_data_ptr<float>(),
                                       grad.const_data_ptr<float>(), grad.dim() == 0 ? 0 : grad.stride(0),
                                       static_cast<const float*>(in_ptr(scale)), out_ptr(dx), ldd, stream_of(logits)));
            out[0] = dx;
        }
        close(out, grad);
        return out;
    }
};

Tensor topk_distill(const OptTensor& logits_, const OptTensor& idx_, const OptTensor& top_, const OptTensor& lse_, double temperature,
                    double own_temperature, int64_t reduction) {
    no_recorder();
    const Tensor logits = on_gpu(logits_, "logits");
    dtype_code(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits need at least one class");
    const at::IntArrayRef rows = logits.sizes().slice(0, logits.dim() - 1);
    Tensor idx = on_gpu(idx_, "teacher_idx", logits), top = on_gpu(top_, "teacher_logits", logits),
           lse = lse_.has_value() ? on_gpu(lse_, "teacher_lse", logits) : Tensor();
    no_tangent(logits_, "logits"), no_tangent(top_, "teacher_logits"), no_tangent(lse_, "teacher_lse");
    TORCH_CHECK_TYPE(at::isIntegralType(idx.scalar_type(), false), "teacher_idx must hold whole numbers, not ", idx.scalar_type());
    TORCH_CHECK_TYPE(at::isFloatingType(top.scalar_type()), "teacher_logits must not be ", top.scalar_type());
    TORCH_CHECK_TYPE(!lse.defined() || at::isFloatingType(lse.scalar_type()), "teacher_lse must not be ", lse.scalar_type());
    TORCH_CHECK_VALUE(!top.requires_grad() && !(lse.defined() && lse.requires_grad()),
                      "the teacher requires a gradient, which there is none of: detach it");
    TORCH_CHECK_VALUE(idx.dim() == logits.dim() && idx.sizes().slice(0, idx.dim() - 1) == rows && top.sizes() == idx.sizes(),
                      "teacher_idx and teacher_logits need one row of k entries per row of logits: ", logits.sizes(), ", ", idx.sizes(), ", ",
                      top.sizes());
    const int64_t k = idx.size(-1);
    TORCH_CHECK_VALUE(k >= 1 && k <= SCMIAC_DISTILL_MAX_K, "k=", k, " outside 1..", SCMIAC_DISTILL_MAX_K);
    TORCH_CHECK_VALUE(!lse.defined() || lse.sizes() == rows, "teacher_lse needs shape ", rows, ", not ", lse.sizes());
    const c10::DeviceGuard guard(logits.device());
    // of numbers that 32 bits do not hold, what is no class stays none (unsigned ones from 2^63 on are negative in 64 bits)
    if (idx.scalar_type() == at::kUInt64) idx = idx.to(at::kLong), idx = idx.masked_fill(idx.lt(0), 2147483647);
    if (idx.scalar_type() == at::kUInt32) idx = idx.to(at::kLong);
    if (idx.scalar_type() == at::kLong) idx = idx.clamp(-2, 2147483647);
    idx = idx.to(at::kInt).reshape({-1, k}).contiguous();
    top = top.reshape({-1, k}).to(at::kFloat).contiguous();
    if (lse.defined()) lse = lse.reshape({-1}).to(at::kFloat).contiguous();
    const Tensor x = logits.dim() == 2 ? logits : logits.reshape({-1, logits.size(-1)});
    const Tensor loss = at::GradMode::is_enabled() && logits.requires_grad()
                            ? TopkDistill::apply(x, idx, top, given(lse), temperature, own_temperature, reduction)
                            : std::get<0>(distill_forward(x, {idx, top, lse, temperature, own_temperature}, reduction));
    return reduction == SCMIAC_REDUCE_NONE && logits.dim() != 2 ? loss.view(rows) : loss;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    m.def("bind", &bind);
    m.def("linear_act", &linear_act, py::call_guard<py::gil_scoped_release>());
    m.def("top_logits", &top_logits, py::call_guard<py::gil_scoped_release>());
    m.def("topk_distill", &topk_distill, py::call_guard<py::gil_scoped_release>());
}
