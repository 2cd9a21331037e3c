// mws_torch.cpp -- the torch side of the sequence operators: argument checks, outputs and scratch memory from torch's allocator,
// the current stream, and the autograd functions, on top of the C ABI in include/mwseq.h.  In C++ because the smallest calls (one
// action of 50 environments) are bound by the host: a call costs 4 us here and 14 us through ctypes, a recorded forward and backward
// pass 36 us and 143 us (layer norm of 50 x 256).
#include <torch/extension.h>
#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include "../../include/mwseq.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

Tensor given(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }       // what an autograd function takes for "none"

// ---- checks ----
std::string shape_of(at::IntArrayRef s) {
    std::ostringstream o;
    o << "(";
    for (size_t i = 0; i < s.size(); i++) o << (i ? ", " : "") << s[i];
    o << ")";
    return o.str();
}
int type_of(at::ScalarType t) { return t == at::kFloat ? MWS_F32 : t == at::kBFloat16 ? MWS_BF16 : t == at::kHalf ? MWS_F16 : -1; }

// a recording of torch's own operations has the memory of the outputs and not the kernels that fill it
void want_untraced() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    const bool traced = at::tracer::impl::is_dispatch_enabled() || (Modes::any_modes_set() && Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
    TORCH_CHECK(!traced, "the sequence operators cannot be traced (torch.jit.trace, torch.fx): a trace would hold their outputs' memory without the kernels that fill it");
}
void want_activations(const char *what, const Tensor &t, int64_t dims = -1) {
    TORCH_CHECK_TYPE(t.defined(), what, " has to be a tensor");
    TORCH_CHECK_TYPE(type_of(t.scalar_type()) >= 0, what, " is ", t.scalar_type(), ": float32, bfloat16 and float16 are supported");
    TORCH_CHECK_VALUE(dims < 0 || t.dim() == dims, what, " has ", t.dim(), " dimensions, ", dims, " are wanted");
    TORCH_CHECK_VALUE(t.dim() > 0, what, " has no dimension");
    TORCH_CHECK_VALUE(t.size(-1) >= 1, what, " has no channels");
}
void want(const char *what, const Tensor &t, at::IntArrayRef shape, at::ScalarType type, const Tensor &like, std::optional<at::ScalarType> other = std::nullopt) {
    if (!t.defined()) return;
    TORCH_CHECK_VALUE(t.sizes() == shape, what, " has shape ", shape_of(t.sizes()), ", ", shape_of(shape), " is wanted");
    TORCH_CHECK_TYPE(t.scalar_type() == type || (other && t.scalar_type() == *other), what, " is ", t.scalar_type(), ", ", type, " is wanted");
    TORCH_CHECK_VALUE(t.device() == like.device(), what, " is on ", t.device(), ", ", like.device(), " is wanted");
}
void want_gpu(const char *what, const Tensor &t) { TORCH_CHECK_VALUE(t.is_cuda(), what, " is on ", t.device(), ": the kernels run on a GPU and there is no CPU fallback"); }
void want_state(const char *what, const Tensor &t) {
    TORCH_CHECK_TYPE(t.defined(), what, ": state has to be a tensor");
    TORCH_CHECK_VALUE(t.is_contiguous() && !t.is_neg(), "state has to be contiguous: it is updated in place");
}
void want_tokens(const Tensor &x, bool time, const Tensor &reset, const Tensor &lengths) {
    if (reset.defined()) {
        bool fits = time ? reset.dim() == 2 && reset.size(0) == x.size(0) && reset.size(1) == x.size(1) : reset.dim() == 1 && reset.size(0) == x.size(0);
        TORCH_CHECK_VALUE(fits, "reset has shape ", shape_of(reset.sizes()), ", ", shape_of(x.sizes().slice(0, time ? 2 : 1)), " is wanted");
        TORCH_CHECK_TYPE(reset.scalar_type() == at::kBool || reset.scalar_type() == at::kByte, "reset is ", reset.scalar_type(), ", bool or uint8 is wanted");
        TORCH_CHECK_VALUE(reset.device() == x.device(), "reset is on ", reset.device(), ", ", x.device(), " is wanted");
    }
    want("lengths", lengths, x.sizes().slice(0, 1), at::kInt, x);
}

// ---- launches ----
// (a lazily negated view's memory holds the values without their sign)
Tensor rows(const Tensor &t) { return !t.defined() || ((t.stride(-1) == 1 || t.size(-1) == 1) && !t.is_neg()) ? t : t.resolve_neg().contiguous(); }
Tensor dense(const Tensor &t) { return t.defined() ? t.resolve_neg().contiguous() : t; }
Tensor near(const Tensor &t) { return !t.defined() || (t.dim() == 3 && t.stride(1) > MWS_SCAN_MAX_STRIDE) ? dense(t) : rows(t); }
Tensor like(const Tensor &t) { return t.defined() ? at::empty(t.sizes(), t.options()) : t; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
const float *floats(const Tensor &t) { return (const float *)ptr(t); }
int64_t step0(const Tensor &t) { return t.defined() ? t.stride(0) : 0; }
int64_t step1(const Tensor &t) { return t.defined() && t.dim() > 1 ? t.stride(1) : 0; }

int64_t good(int64_t code) {
    TORCH_CHECK(code >= 0, "mwseq: ", mws_last_error());
    return code;
}
template <class F, class A> void launch(F f, const A &a, const Tensor &x) {
    c10::DeviceGuard guard(x.device());
    good(f(&a, c10::hip::getCurrentHIPStream(x.device().index()).stream()));
}
Tensor scratch(int64_t bytes, const Tensor &x) { return at::empty({bytes}, x.options().dtype(at::kByte)); }

// whether derivatives are asked for: backward ones, or forward ones, which the autograd functions refuse
bool records(std::initializer_list<Tensor> all) {
    const bool grads = at::GradMode::is_enabled();
    for (const Tensor &t : all)
        if (t.defined() && ((grads && t.requires_grad()) || t._fw_grad(0).defined())) return true;
    return false;
}
void want_acting(const char *what, std::initializer_list<Tensor> all) {
    TORCH_CHECK(!records(all), what, " has no gradient and updates the state in place: call it under torch.no_grad()");
}
void updated(const Tensor &state) {
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
}
void want_once() {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the sequence operators are once differentiable: create_graph=True is not supported");
}
int64_t needs(std::initializer_list<Tensor> all) {
    int64_t mask = 0, bit = 1;
    for (const Tensor &t : all) {
        if (t.defined() && t.requires_grad()) mask |= bit;
        bit <<= 1;
    }
    return mask;
}

// ---- layer norm ----
mws_norm_args norm_args(const Tensor &flat, const Tensor &weight, const Tensor &bias, double eps) {
    mws_norm_args a = {};
    a.x = ptr(flat), a.weight = ptr(weight), a.bias = ptr(bias);
    a.rows = flat.size(0), a.x_stride = flat.stride(0), a.width = (int32_t)flat.size(1), a.type = type_of(flat.scalar_type());
    a.param_type = weight.defined() ? type_of(weight.scalar_type()) : bias.defined() ? type_of(bias.scalar_type()) : MWS_F32;
    a.eps = (float)eps;
    return a;
}
Tensor flat_rows(const Tensor &x) { return rows(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)})); }
Tensor norm_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, double eps) {
    Tensor flat = flat_rows(x), y = at::empty(x.sizes(), x.options());
    mws_norm_args a = norm_args(flat, weight, bias, eps);
    a.y = ptr(y);
    launch(mws_norm_forward, a, x);
    return y;
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Maybe &weight_, const Maybe &bias_, double eps, int64_t need) {
        Tensor weight = given(weight_), bias = given(bias_);
        ctx->save_for_backward({x, weight, bias});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["need"] = need;
        return norm_forward(x, weight, bias, eps);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        want_once();
        auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2];
        int64_t need = ctx->saved_data["need"].toInt();
        Tensor flat = flat_rows(x), dy = flat_rows(grads[0]);
        Tensor dx = need & 1 ? like(x) : Tensor(), dweight = need & 2 ? like(weight) : Tensor(), dbias = need & 4 ? like(bias) : Tensor();
        mws_norm_args a = norm_args(flat, weight, bias, ctx->saved_data["eps"].toDouble());
        a.dy = ptr(dy), a.dy_stride = dy.stride(0), a.dx = ptr(dx), a.dweight = ptr(dweight), a.dbias = ptr(dbias);
        Tensor space = scratch(a.workspace_bytes = good(mws_norm_workspace(&a)), x);
        a.workspace = ptr(space);
        launch(mws_norm_backward, a, x);
        return {dx, dweight, dbias, Tensor(), Tensor()};
    }
};
Tensor layer_norm(const Tensor &x, const Maybe &weight_, const Maybe &bias_, double eps) {
    want_untraced();
    Tensor weight = given(weight_), bias = given(bias_);
    want_activations("x", x);
    int64_t width = x.size(-1);
    TORCH_CHECK_VALUE(width <= MWS_NORM_MAX_WIDTH, "x is ", width, " wide: ", MWS_NORM_MAX_WIDTH, " is the most");
    want("weight", weight, width, at::kFloat, x, x.scalar_type());
    want("bias", bias, width, at::kFloat, x, x.scalar_type());
    TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "weight is ", weight.scalar_type(), " and bias ", bias.scalar_type(), ": one type is wanted");
    TORCH_CHECK_VALUE(eps >= 0, "eps is ", eps, ": it must not be negative");
    want_gpu("x", x);
    weight = rows(weight), bias = rows(bias);
    return records({x, weight, bias}) ? LayerNorm::apply(x, maybe(weight), maybe(bias), eps, needs({x, weight, bias})) : norm_forward(x, weight, bias, eps);
}

// ---- the short causal convolution ----
mws_conv_args conv_args(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, const Tensor &reset, const Tensor &lengths) {
    mws_conv_args a = {};
    bool step = x.dim() == 2;
    a.x = ptr(x), a.weight = ptr(weight), a.bias = ptr(bias), a.state = ptr(state), a.reset = (const uint8_t *)ptr(reset), a.lengths = (const int32_t *)ptr(lengths);
    a.batch = x.size(0), a.length = step ? 1 : x.size(1);
    a.x_batch = x.stride(0), a.x_time = step ? 0 : x.stride(1), a.reset_batch = step0(reset), a.reset_time = step1(reset);
    a.width = (int32_t)weight.size(0), a.taps = (int32_t)weight.size(1), a.type = type_of(x.scalar_type()), a.param_type = type_of(weight.scalar_type());
    return a;
}
variable_list conv_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, const Tensor &reset, const Tensor &lengths) {
    Tensor y = at::empty(x.sizes(), x.options()), last = at::empty({x.size(0), weight.size(1) - 1, x.size(2)}, x.options());
    mws_conv_args a = conv_args(x, weight, bias, state, reset, lengths);
    a.y = ptr(y), a.last = ptr(last);
    launch(mws_conv_forward, a, x);
    return {y, last};
}
struct CausalConv : torch::autograd::Function<CausalConv> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Maybe &bias_, const Maybe &state_, const Maybe &reset_, const Maybe &lengths_, int64_t need) {
        Tensor bias = given(bias_), state = given(state_), reset = given(reset_), lengths = given(lengths_);
        ctx->save_for_backward({x, weight, bias, state, reset, lengths});
        ctx->saved_data["need"] = need;
        ctx->set_materialize_grads(false);
        return conv_forward(x, weight, bias, state, reset, lengths);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        want_once();
        auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &weight = s[1], &bias = s[2], &state = s[3];
        int64_t need = ctx->saved_data["need"].toInt();
        Tensor dy = grads[0].defined() ? rows(grads[0]) : at::zeros(x.sizes(), x.options()), dlast = dense(grads[1]);
        Tensor dx = need & 1 ? like(x) : Tensor(), dweight = need & 2 ? like(weight) : Tensor(), dbias = need & 4 ? like(bias) : Tensor(), dstate = need & 8 ? like(state) : Tensor();
        mws_conv_args a = conv_args(x, weight, bias, state, s[4], s[5]);
        a.dy = ptr(dy), a.dy_batch = dy.stride(0), a.dy_time = dy.stride(1), a.dlast = ptr(dlast);
        a.dx = ptr(dx), a.dweight = ptr(dweight), a.dbias = ptr(dbias), a.dstate = ptr(dstate);
        Tensor space = scratch(a.workspace_bytes = good(mws_conv_workspace(&a)), x);
        a.workspace = ptr(space);
        launch(mws_conv_backward, a, x);
        return {dx, dweight, dbias, dstate, Tensor(), Tensor(), Tensor()};
    }
};
void conv_check(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, int64_t dims) {
    want_activations("x", x, dims);
    int64_t width = x.size(-1);
    TORCH_CHECK_TYPE(weight.scalar_type() == at::kFloat || weight.scalar_type() == x.scalar_type(), "weight is ", weight.scalar_type(), ", float32 or ", x.scalar_type(), " is wanted");
    TORCH_CHECK_VALUE(weight.device() == x.device(), "weight is on ", weight.device(), ", ", x.device(), " is wanted");
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) == width && weight.size(1) >= MWS_CONV_MIN_TAPS && weight.size(1) <= MWS_CONV_MAX_TAPS, "weight has shape ", shape_of(weight.sizes()),
                      ", (", width, ", ", MWS_CONV_MIN_TAPS, " .. ", MWS_CONV_MAX_TAPS, " taps) is wanted");
    want("bias", bias, width, weight.scalar_type(), x);
    want("state", state, {x.size(0), weight.size(1) - 1, width}, x.scalar_type(), x);
}
variable_list causal_conv(Tensor x, Tensor weight, const Maybe &bias_, const Maybe &state_, const Maybe &reset_, const Maybe &lengths_) {
    want_untraced();
    Tensor bias = given(bias_), state = given(state_), reset = given(reset_), lengths = given(lengths_);
    conv_check(x, weight, bias, state, 3);
    want_tokens(x, true, reset, lengths);
    want_gpu("x", x);
    x = rows(x), weight = dense(weight), bias = rows(bias), state = dense(state), lengths = dense(lengths);
    return records({x, weight, bias, state}) ? CausalConv::apply(x, weight, maybe(bias), maybe(state), maybe(reset), maybe(lengths), needs({x, weight, bias, state})) : conv_forward(x, weight, bias, state, reset, lengths);
}
Tensor causal_conv_step(Tensor x, Tensor weight, const Maybe &bias_, const Maybe &state_, const Maybe &reset_) {
    want_untraced();
    Tensor bias = given(bias_), state = given(state_), reset = given(reset_);
    conv_check(x, weight, bias, state, 2);
    want_tokens(x, false, reset, Tensor());
    want_state("causal_conv_step", state);
    want_gpu("x", x);
    want_acting("causal_conv_step", {x, weight, bias, state});
    x = rows(x), weight = dense(weight), bias = rows(bias);
    Tensor y = at::empty(x.sizes(), x.options());
    mws_conv_args a = conv_args(x, weight, bias, state, reset, Tensor());
    a.y = ptr(y), a.last = ptr(state);
    launch(mws_conv_step, a, x);
    updated(state);
    return y;
}

// ---- the selective state space scan ----
struct ScanIn {
    Tensor u, dt, A, B, C, D, z, dt_bias, state, reset, lengths;
};
mws_scan_args scan_args(const ScanIn &t) {
    mws_scan_args a = {};
    bool step = t.u.dim() == 2;
    a.u = ptr(t.u), a.dt = ptr(t.dt), a.z = ptr(t.z), a.B = ptr(t.B), a.C = ptr(t.C);
    a.A = floats(t.A), a.D = floats(t.D), a.dt_bias = floats(t.dt_bias), a.state = floats(t.state);
    a.reset = (const uint8_t *)ptr(t.reset), a.lengths = (const int32_t *)ptr(t.lengths);
    a.batch = t.u.size(0), a.length = step ? 1 : t.u.size(1);
    a.u_batch = step0(t.u), a.dt_batch = step0(t.dt), a.z_batch = step0(t.z), a.B_batch = step0(t.B), a.C_batch = step0(t.C), a.reset_batch = step0(t.reset);
    if (!step) a.u_time = step1(t.u), a.dt_time = step1(t.dt), a.z_time = step1(t.z), a.B_time = step1(t.B), a.C_time = step1(t.C), a.reset_time = step1(t.reset);
    a.width = (int32_t)t.A.size(0), a.states = (int32_t)t.A.size(1), a.type = type_of(t.u.scalar_type());
    return a;
}
variable_list scan_forward(const ScanIn &t, bool keep) {
    auto wide = t.u.options().dtype(at::kFloat);
    Tensor y = at::empty(t.u.sizes(), t.u.options()), last = at::empty({t.u.size(0), t.A.size(0), t.A.size(1)}, wide), kept;
    mws_scan_args a = scan_args(t);
    a.y = ptr(y), a.last = (float *)ptr(last);
    if (keep) {
        kept = at::empty({good(mws_scan_kept(&a))}, wide);
        a.kept = (float *)ptr(kept);
    }
    Tensor space = scratch(a.workspace_bytes = good(mws_scan_workspace(&a, 0)), t.u);
    a.workspace = ptr(space);
    launch(mws_scan_forward, a, t.u);
    return {y, last, kept};
}
struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &u, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Maybe &D, const Maybe &z, const Maybe &dt_bias,
                                 const Maybe &state, const Maybe &reset, const Maybe &lengths) {
        ScanIn t = {u, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(reset), given(lengths)};
        variable_list out = scan_forward(t, true);
        ctx->save_for_backward({u, dt, A, B, C, t.D, t.z, t.dt_bias, t.state, t.reset, t.lengths, out[2]});
        ctx->set_materialize_grads(false);
        return {out[0], out[1]};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        want_once();
        auto s = ctx->get_saved_variables();
        ScanIn t = {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], s[10]};
        Tensor dy = grads[0].defined() ? near(grads[0]) : at::zeros(t.u.sizes(), t.u.options()), dlast = dense(grads[1]);
        variable_list d;
        for (int k = 0; k < 9; k++) d.push_back(like(s[k]));
        mws_scan_args a = scan_args(t);
        a.dy = ptr(dy), a.dy_batch = dy.stride(0), a.dy_time = dy.stride(1), a.dlast = floats(dlast), a.kept = (float *)ptr(s[11]);
        a.du = ptr(d[0]), a.ddt = ptr(d[1]), a.dA = (float *)ptr(d[2]), a.dB = ptr(d[3]), a.dC = ptr(d[4]), a.dD = (float *)ptr(d[5]), a.dz = ptr(d[6]);
        a.ddt_bias = (float *)ptr(d[7]), a.dstate = (float *)ptr(d[8]);
        Tensor space = scratch(a.workspace_bytes = good(mws_scan_workspace(&a, 1)), t.u);
        a.workspace = ptr(space);
        launch(mws_scan_backward, a, t.u);
        d.resize(11);
        return d;
    }
};
ScanIn scan_check(const Tensor &u, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Maybe &D, const Maybe &z, const Maybe &dt_bias, const Maybe &state, const Maybe &reset,
                  const Maybe &lengths, int64_t dims) {
    want_untraced();
    ScanIn t = {u, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(reset), given(lengths)};
    want_activations("u", u, dims);
    int64_t width = u.size(-1);
    TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == width && A.size(1) >= 1 && A.size(1) <= MWS_SCAN_MAX_STATES, "A has shape ", shape_of(A.sizes()), ", (", width, ", 1 .. ",
                      MWS_SCAN_MAX_STATES, " states) is wanted");
    want("A", A, A.sizes(), at::kFloat, u);
    want("dt", dt, u.sizes(), u.scalar_type(), u);
    want("z", t.z, u.sizes(), u.scalar_type(), u);
    std::vector<int64_t> shared = u.sizes().vec();
    shared.back() = A.size(1);
    want("B", B, shared, u.scalar_type(), u);
    want("C", C, shared, u.scalar_type(), u);
    want("D", t.D, width, at::kFloat, u);
    want("dt_bias", t.dt_bias, width, at::kFloat, u);
    want("state", t.state, {u.size(0), width, A.size(1)}, at::kFloat, u);
    want_tokens(u, dims == 3, t.reset, t.lengths);
    return t;
}
void scan_rows(ScanIn &t) {
    t.u = near(t.u), t.dt = near(t.dt), t.B = rows(t.B), t.C = rows(t.C), t.D = rows(t.D), t.z = near(t.z), t.dt_bias = rows(t.dt_bias), t.A = dense(t.A);
}
variable_list selective_scan(const Tensor &u, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Maybe &D, const Maybe &z, const Maybe &dt_bias, const Maybe &state,
                             const Maybe &reset, const Maybe &lengths) {
    ScanIn t = scan_check(u, dt, A, B, C, D, z, dt_bias, state, reset, lengths, 3);
    want_gpu("u", u);
    scan_rows(t);
    t.state = dense(t.state), t.lengths = dense(t.lengths);
    if (records({t.u, t.dt, t.A, t.B, t.C, t.D, t.z, t.dt_bias, t.state})) return SelectiveScan::apply(t.u, t.dt, t.A, t.B, t.C, maybe(t.D), maybe(t.z), maybe(t.dt_bias), maybe(t.state), maybe(t.reset), maybe(t.lengths));
    variable_list out = scan_forward(t, false);
    out.pop_back();
    return out;
}
Tensor selective_scan_step(const Tensor &u, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Maybe &D, const Maybe &z, const Maybe &dt_bias, const Maybe &state,
                           const Maybe &reset) {
    ScanIn t = scan_check(u, dt, A, B, C, D, z, dt_bias, state, reset, std::nullopt, 2);
    want_state("selective_scan_step", t.state);
    want_gpu("u", u);
    want_acting("selective_scan_step", {t.u, t.dt, t.A, t.B, t.C, t.D, t.z, t.dt_bias, t.state});
    scan_rows(t);
    Tensor y = at::empty(u.sizes(), u.options());
    mws_scan_args a = scan_args(t);
    a.y = ptr(y), a.last = (float *)ptr(t.state);
    launch(mws_scan_step, a, t.u);
    updated(t.state);
    return y;
}
}  // namespace

PYBIND11_MODULE(_sequence, m) {
    m.def("layer_norm", &layer_norm);
    m.def("causal_conv", [](Tensor x, Tensor w, const Maybe &b, const Maybe &s, const Maybe &r, const Maybe &l) {
        variable_list o = causal_conv(x, w, b, s, r, l);
        return std::make_pair(o[0], o[1]);
    });
    m.def("causal_conv_step", &causal_conv_step);
    m.def("selective_scan", [](const Tensor &u, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Maybe &D, const Maybe &z, const Maybe &bias, const Maybe &s,
                               const Maybe &r, const Maybe &l) {
        variable_list o = selective_scan(u, dt, A, B, C, D, z, bias, s, r, l);
        return std::make_pair(o[0], o[1]);
    });
    m.def("selective_scan_step", &selective_scan_step);
}
