// otf_torch.cpp — the fusion block's layers as autograd nodes over the C ABI (include/otfuse.h).
//
// This module checks the arguments of otfuse/layers.py's functions, allocates the results, calls
// libotfuse.so on the current stream of the tensors' device, and records backward.  Native rather
// than Python because the layers' smallest calls are bound by the host: a trained dropout of 8 x 512
// float32 took 107 us as a torch.autograd.Function in Python, whose backward has to take the
// interpreter lock on the engine's thread, against 4 us of kernels (47 us here); a norm of one token
// 16 us, 7 with the checks in Python.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "otfuse.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct OtfFailure : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc, const char* what) {
    if (rc == OTF_OK) return;
    const char* kind = rc == OTF_EINVAL ? "invalid argument" : rc == OTF_EUNSUPPORTED ? "unsupported shape/config"
                       : rc == OTF_EHIP ? "HIP runtime error" : "error";
    throw OtfFailure(std::string(what) + ": " + kind + " (rc=" + std::to_string(rc) + ")");
}

int32_t type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return OTF_F32;
        case at::kHalf: return OTF_F16;
        case at::kBFloat16: return OTF_BF16;
        default: throw OtfFailure("float32, bfloat16 or float16 tensors only");
    }
}

otf_stream_t stream_of(const Tensor& t) {
    return (otf_stream_t)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

// a lazily negated view (the imaginary part of a conjugate) as the values that it stands for
Tensor resolved(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
// (..., cols) -> (rows, cols) with unit column stride and rows that do not overlap
Tensor rows_of(const Tensor& t, int64_t cols) {
    const Tensor r = resolved(t.dim() == 2 ? t : t.reshape({-1, cols}));
    return r.stride(1) == 1 && r.stride(0) >= cols ? r : r.contiguous();
}
// A single row has no leading dimension, whatever its stride (contiguous() keeps any): its columns.
int64_t ld(const Tensor& t) { return !t.defined() ? 0 : t.size(0) <= 1 ? t.size(1) : std::max(t.stride(0), t.size(1)); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor dense(const OptTensor& t) { return t.has_value() && t->defined() ? resolved(*t).contiguous() : Tensor(); }
const int64_t* words(const Tensor& rng) { return rng.defined() ? rng.const_data_ptr<int64_t>() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const OptTensor& t) { return t.has_value() && wants(*t); }

// ---- what every entry point refuses (TypeError, ValueError) --------------------------------
std::string text(const Tensor& t) {
    std::ostringstream o;
    o << t.sizes() << " " << t.scalar_type();
    return o.str();
}
// What the kernels would drop without a word: a tangent of forward-mode differentiation, and themselves
// from a trace, which would hold the allocation of the results alone (RuntimeError)
void plain(const Tensor& t, const char* name) {
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
        throw OtfFailure(std::string(name) + " carries a forward-mode tangent: the layers have reverse mode only");
}
void no_trace() {
    if (torch::jit::tracer::isTracing()) throw OtfFailure("the layers cannot be traced: a trace would not hold their kernels");
}
void input(const Tensor& t, const char* name) {
    if (!t.defined() || !t.is_cuda()) throw py::type_error(std::string(name) + " must be a ROCm device tensor");
    const auto k = t.scalar_type();
    if (k != at::kFloat && k != at::kHalf && k != at::kBFloat16)
        throw py::type_error(std::string(name) + ": float32, bfloat16 or float16, not " + text(t));
    plain(t, name);
}
void beside(const Tensor& x, const Tensor& t, const char* name) {
    if (t.device() != x.device()) throw py::value_error(std::string(name) + " is not on x's device");
}
double probability(double p) {
    if (!(p >= 0.0 && p <= 1.0)) throw py::value_error("dropout probability " + std::to_string(p) + " is not in [0, 1]");
    return p;
}
double epsilon(double eps) {
    if (!(eps >= 0.0 && eps < std::numeric_limits<double>::infinity()))
        throw py::value_error("eps " + std::to_string(eps) + " must be finite and not negative");
    return eps;
}
void state(const Tensor& rng, const Tensor& x) {
    if (rng.scalar_type() != at::kLong || rng.dim() != 1 || rng.size(0) != 2 || !rng.is_contiguous())
        throw py::type_error("rng must be a contiguous int64 tensor [seed, offset] (rng_state)");
    beside(x, rng, "rng");
}
void norm_params(const Tensor& x, const OptTensor& weight, const OptTensor& bias) {
    if (x.dim() == 0 || x.size(-1) == 0) throw py::value_error("x " + text(x) + ": layer norm needs a last dimension of at least 1");
    const OptTensor* both[2] = {&weight, &bias};
    for (int i = 0; i < 2; ++i) {
        if (!both[i]->has_value()) continue;
        const Tensor& t = **both[i];
        const char* name = i ? "bias" : "weight";
        input(t, name);
        beside(x, t, name);
        if (t.dim() != 1 || t.size(0) != x.size(-1)) throw py::value_error(std::string(name) + " " + text(t) + " must have x's columns");
        if (t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat)
            throw py::type_error(std::string(name) + " must have x's type or float32, not " + text(t));
    }
    if (weight.has_value() && bias.has_value() && weight->scalar_type() != bias->scalar_type())
        throw py::type_error("weight and bias must share one type");
}

// Gradients of kernels are not differentiable: under create_graph they carry a node that says so
// when it is reached.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    torch::autograd::DelayedError error("trying to differentiate twice a layer whose backward is a kernel", (int64_t)grads.size());
    return error.apply(std::move(grads));
}

// ------------------------------------------------------------------------------- dropout
Tensor dropout_call(const Tensor& x, const Tensor& residual, double p, const Tensor& rng) {
    if (x.numel() == 0) return at::empty(x.sizes(), x.options());
    const c10::DeviceGuard guard(x.device());
    const int64_t cols = x.dim() ? x.size(-1) : 1;
    const Tensor x2 = rows_of(x, cols), r2 = residual.defined() ? rows_of(residual, cols) : Tensor();
    Tensor y = at::empty(x.sizes(), x.options());
    check(otf_dropout(ptr(x2), ld(x2), ptr(r2), ld(r2), ptr(y), cols, x2.size(0), cols, type_of(x), p,
                      words(rng), stream_of(x)),
          "otf_dropout");
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, double p, const Tensor& rng) {
        ctx->save_for_backward({rng});
        ctx->saved_data["p"] = p;
        ctx->saved_data["x"] = wants(x);
        ctx->saved_data["residual"] = wants(residual);
        return dropout_call(x, value(residual), p, rng);
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        plain(dy[0], "a gradient");
        const auto rng = ctx->get_saved_variables()[0];
        variable_list g(4);
        if (ctx->saved_data["x"].toBool()) g[0] = dropout_call(dy[0], Tensor(), ctx->saved_data["p"].toDouble(), rng);
        if (ctx->saved_data["residual"].toBool()) g[1] = dy[0];
        return once(std::move(g));
    }
};

Tensor dropout(const Tensor& x, double p, const Tensor& rng, const OptTensor& residual) {
    no_trace();
    input(x, "x");
    if (residual.has_value()) {
        input(*residual, "residual");
        beside(x, *residual, "residual");
        if (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type())
            throw py::value_error("residual " + text(*residual) + " differs from x " + text(x));
    }
    probability(p);
    state(rng, x);
    if (at::GradMode::is_enabled() && (wants(x) || wants(residual))) return Dropout::apply(x, residual, p, rng);
    return dropout_call(x, value(residual), p, rng);
}

// ---------------------------------------------------------------------------- layer norm
// the type that weight and bias share
int32_t param_type(const OptTensor& w, const OptTensor& b) {
    return w.has_value() ? type_of(*w) : b.has_value() ? type_of(*b) : OTF_F32;
}
Tensor stats_of(int64_t rows, const Tensor& x) { return at::empty({2, rows}, x.options().dtype(at::kFloat)); }
float* stat(const Tensor& s, int which) { return s.defined() ? s.data_ptr<float>() + which * s.size(1) : nullptr; }

struct ParamGrads {
    Tensor dw, db, ws;
};
ParamGrads param_grads(const Tensor& like, int64_t rows, int64_t cols, int32_t type, bool w, bool b) {
    ParamGrads g;
    const auto t = type == OTF_F32 ? at::kFloat : type == OTF_F16 ? at::kHalf : at::kBFloat16;
    if (w) g.dw = at::empty({cols}, like.options().dtype(t));
    if (b) g.db = at::empty({cols}, like.options().dtype(t));
    const size_t size = w || b ? otf_layer_norm_backward_workspace_size(rows, cols) : 0;
    if (size) g.ws = at::empty({(int64_t)size}, like.options().dtype(at::kByte));
    return g;
}
size_t bytes_of(const Tensor& t) { return t.defined() ? (size_t)t.numel() : 0; }

Tensor layer_norm_call(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, const Tensor& x2,
                       const Tensor& stats) {
    const int64_t cols = x.size(-1);
    const Tensor w = dense(weight), b = dense(bias);
    Tensor y = at::empty(x.sizes(), x.options());
    check(otf_layer_norm(ptr(x2), ld(x2), type_of(x), ptr(w), ptr(b), param_type(weight, bias), eps, x2.size(0), cols,
                         ptr(y), cols, stat(stats, 0), stat(stats, 1), stream_of(x)),
          "otf_layer_norm");
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
        const c10::DeviceGuard guard(x.device());
        const Tensor x2 = rows_of(x, x.size(-1)), stats = stats_of(x2.size(0), x);
        // a copied row layout is kept as copied; else the input itself, so that a change of it before
        // backward is noticed
        ctx->save_for_backward({x2.const_data_ptr() == x.const_data_ptr() ? x : x2, value(weight), stats});
        ctx->saved_data["type"] = (int64_t)param_type(weight, bias);
        ctx->saved_data["x"] = wants(x);
        ctx->saved_data["w"] = wants(weight);
        ctx->saved_data["b"] = wants(bias);
        return layer_norm_call(x, weight, bias, eps, x2, stats);
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        plain(dy[0], "a gradient");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &stats = saved[2];
        const int64_t cols = x.size(-1);
        const int32_t type = (int32_t)ctx->saved_data["type"].toInt();
        const bool want_w = ctx->saved_data["w"].toBool(), want_b = ctx->saved_data["b"].toBool();
        const c10::DeviceGuard guard(stats.device());
        const Tensor x2 = rows_of(x, cols), dy2 = rows_of(dy[0], cols), w = dense(saved[1]);
        Tensor dx = at::empty(dy[0].sizes(), x.options());
        const ParamGrads p = param_grads(x, x2.size(0), cols, type, want_w, want_b);
        check(otf_layer_norm_backward(ptr(dy2), ld(dy2), ptr(x2), ld(x2), type_of(x), ptr(w), type, stat(stats, 0),
                                      stat(stats, 1), x2.size(0), cols, ptr(dx), cols, ptr(p.dw), ptr(p.db), ptr(p.ws),
                                      bytes_of(p.ws), stream_of(x)),
              "otf_layer_norm_backward");
        return once({ctx->saved_data["x"].toBool() ? dx : Tensor(), p.dw, p.db, Tensor()});
    }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    no_trace();
    input(x, "x");
    norm_params(x, weight, bias);
    epsilon(eps);
    if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias)))
        return LayerNorm::apply(x, weight, bias, eps);
    const c10::DeviceGuard guard(x.device());
    return layer_norm_call(x, weight, bias, eps, rows_of(x, x.size(-1)), Tensor());
}

// ------------------------------------------------------------------------- residual norm
std::pair<Tensor, Tensor> add_norm_call(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                        const OptTensor& bias, double p, const Tensor& rng, double eps, const Tensor& x2,
                                        const Tensor& r2, const Tensor& stats) {
    const int64_t cols = x.size(-1);
    const Tensor w = dense(weight), b = dense(bias);
    Tensor y = at::empty(x.sizes(), x.options());
    Tensor z = at::empty(x.sizes(), residual.options());
    check(otf_dropout_add_layer_norm(ptr(x2), ld(x2), type_of(x), ptr(r2), ld(r2), type_of(residual), ptr(w), ptr(b),
                                     param_type(weight, bias), eps, p, words(rng), x2.size(0), cols,
                                     ptr(y), cols, ptr(z), cols, stat(stats, 0), stat(stats, 1), stream_of(x)),
          "otf_dropout_add_layer_norm");
    return {y, z};
}

struct AddNorm : torch::autograd::Function<AddNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                 const OptTensor& bias, double p, const OptTensor& state, double eps) {
        const c10::DeviceGuard guard(x.device());
        const Tensor rng = value(state);
        const int64_t cols = x.size(-1);
        const Tensor x2 = rows_of(x, cols), r2 = rows_of(residual, cols), stats = stats_of(x2.size(0), x);
        auto [y, z] = add_norm_call(x, residual, weight, bias, p, rng, eps, x2, r2, stats);
        ctx->set_materialize_grads(false);
        // a float32 z is the normalised sum itself; a rounded one is not: keep what it is the sum of
        if (z.scalar_type() == at::kFloat)
            ctx->save_for_backward({value(weight), stats, rng, z});
        else
            ctx->save_for_backward({value(weight), stats, rng, x2.const_data_ptr() == x.const_data_ptr() ? x : x2,
                                    r2.const_data_ptr() == residual.const_data_ptr() ? residual : r2});
        ctx->saved_data["type"] = (int64_t)param_type(weight, bias);
        ctx->saved_data["xtype"] = (int64_t)x.scalar_type();
        ctx->saved_data["rtype"] = (int64_t)z.scalar_type();
        ctx->saved_data["p"] = p;
        ctx->saved_data["x"] = wants(x);
        ctx->saved_data["residual"] = wants(residual);
        ctx->saved_data["w"] = wants(weight);
        ctx->saved_data["b"] = wants(bias);
        return {y, z};
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        Tensor dy = d[0];
        const Tensor dz = d[1];
        if (!dy.defined() && !dz.defined()) return variable_list(7);
        for (const Tensor& g : d) plain(g, "a gradient");
        const auto saved = ctx->get_saved_variables();
        const Tensor &stats = saved[1], &rng = saved[2];
        const auto xtype = (at::ScalarType)ctx->saved_data["xtype"].toInt(), rtype = (at::ScalarType)ctx->saved_data["rtype"].toInt();
        const int32_t type = (int32_t)ctx->saved_data["type"].toInt();
        const c10::DeviceGuard guard(stats.device());
        const auto sizes = (dy.defined() ? dy : dz).sizes();
        if (!dy.defined()) dy = at::zeros(sizes, stats.options().dtype(xtype));
        const int64_t rows = stats.size(1), cols = sizes.back();
        const bool again = saved.size() == 5;
        const Tensor z2 = again ? Tensor() : rows_of(saved[3], cols), x2 = again ? rows_of(saved[3], cols) : Tensor();
        const Tensor r2 = again ? rows_of(saved[4], cols) : Tensor();
        const Tensor dy2 = rows_of(dy, cols), dz2 = dz.defined() ? rows_of(dz, cols) : Tensor(), w = dense(saved[0]);
        Tensor dx = at::empty(sizes, stats.options().dtype(xtype)), dr = at::empty(sizes, stats.options().dtype(rtype));
        const ParamGrads g = param_grads(stats, rows, cols, type, ctx->saved_data["w"].toBool(), ctx->saved_data["b"].toBool());
        check(otf_dropout_add_layer_norm_backward(ptr(dy2), ld(dy2), ptr(dz2), ld(dz2), ptr(z2), ld(z2), ptr(x2), ld(x2),
                                                  ptr(r2), ld(r2), type_of(dx), type_of(dr), ptr(w), type, stat(stats, 0),
                                                  stat(stats, 1), ctx->saved_data["p"].toDouble(),
                                                  words(rng), rows, cols, ptr(dx), cols, ptr(dr), cols,
                                                  ptr(g.dw), ptr(g.db), ptr(g.ws), bytes_of(g.ws), stream_of(stats)),
              "otf_dropout_add_layer_norm_backward");
        return once({ctx->saved_data["x"].toBool() ? dx : Tensor(), ctx->saved_data["residual"].toBool() ? dr : Tensor(),
                     g.dw, g.db, Tensor(), Tensor(), Tensor()});
    }
};

std::pair<Tensor, Tensor> dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                                 const OptTensor& bias, double p, const OptTensor& rng, double eps) {
    no_trace();
    input(x, "x");
    input(residual, "residual");
    beside(x, residual, "residual");
    if (residual.sizes() != x.sizes()) throw py::value_error("residual " + text(residual) + " differs from x " + text(x));
    if (residual.scalar_type() != x.scalar_type() && residual.scalar_type() != at::kFloat)
        throw py::type_error("residual must have x's type or float32, not " + text(residual));
    norm_params(x, weight, bias);
    probability(p);
    epsilon(eps);
    if (rng.has_value())
        state(*rng, x);
    else if (p > 0.0)
        throw py::value_error("p > 0 needs rng (rng_state)");
    if (at::GradMode::is_enabled() && (wants(x) || wants(residual) || wants(weight) || wants(bias))) {
        const variable_list o = AddNorm::apply(x, residual, weight, bias, p, rng, eps);
        return {o[0], o[1]};
    }
    const c10::DeviceGuard guard(x.device());
    const int64_t cols = x.size(-1);
    return add_norm_call(x, residual, weight, bias, p, value(rng), eps, rows_of(x, cols), rows_of(residual, cols), Tensor());
}

// -------------------------------------------------------------------- gated feed-forward
constexpr int64_t kMaxLd = 1 << 20;   // the kernels' row strides
Tensor near_rows(const Tensor& t, int64_t cols) {
    const Tensor r = rows_of(t, cols);
    return ld(r) <= kMaxLd ? r : r.contiguous();
}

struct FfnInputs {
    Tensor x, wg, wu, wd;
    otf_ffn_args a{};
    FfnInputs(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const Tensor& wd_, int64_t act) {
        const int64_t d = x_.size(-1), f = wg_.size(0);
        x = near_rows(x_, d), wg = near_rows(wg_, d), wu = near_rows(wu_, d), wd = near_rows(wd_, f);
        if (ld(wg) != ld(wu)) wg = wg.contiguous(), wu = wu.contiguous();   // one leading dimension
        a.rows = x.size(0), a.d = d, a.f = f, a.dtype = type_of(x), a.activation = (int32_t)act;
        a.x = ptr(x), a.ldx = ld(x), a.w_gate = ptr(wg), a.w_up = ptr(wu), a.ldw_in = std::max(ld(wg), ld(wu));
        a.w_down = ptr(wd), a.ldw_down = ld(wd);
    }
};

Tensor ffn_call(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act, Tensor* saved) {
    const c10::DeviceGuard guard(x.device());
    FfnInputs in(x, wg, wu, wd, act);
    otf_ffn_args& a = in.a;
    Tensor y = at::empty(x.sizes(), x.options());
    const auto bytes = x.options().dtype(at::kByte);
    if (saved) *saved = at::empty({(int64_t)otf_gated_ffn_saved_size(a.rows, a.f, a.dtype)}, bytes);
    a.y = ptr(y), a.ldy = a.d, a.saved = saved ? ptr(*saved) : nullptr;
    const size_t size = otf_gated_ffn_workspace_size(&a);
    const Tensor ws = size ? at::empty({(int64_t)size}, bytes) : Tensor();
    check(otf_gated_ffn(&a, ptr(ws), size, stream_of(x)), "otf_gated_ffn");
    return y;
}

struct GatedFeedForward : torch::autograd::Function<GatedFeedForward> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
        Tensor saved;
        Tensor y = ffn_call(x, wg, wu, wd, act, &saved);
        ctx->save_for_backward({x, wg, wu, wd, saved});
        ctx->saved_data["act"] = act;
        ctx->saved_data["x"] = wants(x);
        ctx->saved_data["wg"] = wants(wg);
        ctx->saved_data["wu"] = wants(wu);
        ctx->saved_data["wd"] = wants(wd);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        plain(grads[0], "a gradient");
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &dy = grads[0];
        const c10::DeviceGuard guard(x.device());
        FfnInputs in(x, s[1], s[2], s[3], ctx->saved_data["act"].toInt());
        otf_ffn_args& a = in.a;
        const Tensor dy2 = near_rows(dy, a.d);
        const bool gate = ctx->saved_data["wg"].toBool(), up = ctx->saved_data["wu"].toBool();
        Tensor dx, dwg, dwu, dwd;
        if (ctx->saved_data["x"].toBool()) dx = at::empty(x.sizes(), x.options());
        if (gate || up) dwg = at::empty({a.f, a.d}, x.options()), dwu = at::empty({a.f, a.d}, x.options());   // one product
        if (ctx->saved_data["wd"].toBool()) dwd = at::empty({a.d, a.f}, x.options());
        a.saved = ptr(s[4]), a.dy = ptr(dy2), a.lddy = ld(dy2), a.dx = ptr(dx), a.lddx = a.d;
        a.dw_gate = ptr(dwg), a.dw_up = ptr(dwu), a.lddw_in = a.d, a.dw_down = ptr(dwd), a.lddw_down = a.f;
        const size_t size = otf_gated_ffn_backward_workspace_size(&a);
        const Tensor ws = size ? at::empty({(int64_t)size}, x.options().dtype(at::kByte)) : Tensor();
        check(otf_gated_ffn_backward(&a, ptr(ws), size, stream_of(x)), "otf_gated_ffn_backward");
        return once({dx, gate ? dwg : Tensor(), up ? dwu : Tensor(), dwd, Tensor()});
    }
};

Tensor gated_feed_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const std::string& activation) {
    no_trace();
    input(x, "x");
    const std::pair<const Tensor*, const char*> weights[3] = {{&wg, "w_gate"}, {&wu, "w_up"}, {&wd, "w_down"}};
    for (const auto& [t, name] : weights) {
        input(*t, name);
        beside(x, *t, name);
        if (t->scalar_type() != x.scalar_type()) throw py::type_error(std::string(name) + " " + text(*t) + " must have x's type");
    }
    const int64_t act = activation == "silu" ? OTF_ACT_SILU : activation == "gelu" ? OTF_ACT_GELU : -1;
    if (act < 0) throw py::value_error("activation '" + activation + "': silu or gelu");
    const int64_t d = x.dim() ? x.size(-1) : 0;
    if (wg.dim() != 2 || wg.size(1) != d || wu.sizes() != wg.sizes() || wd.dim() != 2 || wd.size(0) != d || wd.size(1) != wg.size(0))
        throw py::value_error("x " + text(x) + ", w_gate " + text(wg) + ", w_up " + text(wu) + " and w_down " + text(wd) +
                              " must be (..., d), (f, d), (f, d) and (d, f)");
    if (d == 0 || wg.size(0) == 0 || std::max(d, wg.size(0)) > kMaxLd)
        throw py::value_error("widths d = " + std::to_string(d) + " and f = " + std::to_string(wg.size(0)) + " must be between 1 and 2^20");
    if (at::GradMode::is_enabled() && (wants(x) || wants(wg) || wants(wu) || wants(wd)))
        return GatedFeedForward::apply(x, wg, wu, wd, act);
    return ffn_call(x, wg, wu, wd, act, nullptr);
}

}  // namespace

PYBIND11_MODULE(_otf_layers, m) {
    static py::object error = py::module_::import("otfuse._lib").attr("OtfError");
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const OtfFailure& e) {
            PyErr_SetString(error.ptr(), e.what());
        }
    });
    m.def("dropout", &dropout);
    m.def("layer_norm", &layer_norm);
    m.def("dropout_add_layer_norm", &dropout_add_layer_norm);
    m.def("gated_feed_forward", &gated_feed_forward);
}
