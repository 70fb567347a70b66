// The torch side of the sequence-memory and optimizer operators: argument checks, output allocation, and the autograd
// functions over the C entries (include/vsv_hip.h).  Native because a call of theirs takes the GPU a few microseconds: the
// same code in Python took the host 45 us forward and 60 us backward (on top of what autograd itself takes).
// The C entries' addresses come from the library that vsv/lib.py has loaded (bind), so there is one copy of it.
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>

#include "../../include/vsv_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Api {
    decltype(&vsv_short_conv) short_conv;
    decltype(&vsv_short_conv_backward_ws_bytes) short_conv_backward_ws_bytes;
    decltype(&vsv_short_conv_backward) short_conv_backward;
    decltype(&vsv_short_conv_step) short_conv_step;
    decltype(&vsv_ssm_saved_floats) ssm_saved_floats;
    decltype(&vsv_ssm_scan_ws_bytes) ssm_scan_ws_bytes;
    decltype(&vsv_ssm_scan) ssm_scan;
    decltype(&vsv_ssm_scan_backward_ws_bytes) ssm_scan_backward_ws_bytes;
    decltype(&vsv_ssm_scan_backward) ssm_scan_backward;
    decltype(&vsv_ssm_step) ssm_step;
    decltype(&vsv_adamw_multi) adamw_multi;
    decltype(&vsv_adamw_read8) adamw_read8;
    const char* (*last_error)(void);
} api;

void bind(const std::map<std::string, uintptr_t>& at) {
    auto set = [&](auto& fn, const char* name) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at.at(name)); };
    set(api.short_conv, "vsv_short_conv");
    set(api.short_conv_backward_ws_bytes, "vsv_short_conv_backward_ws_bytes");
    set(api.short_conv_backward, "vsv_short_conv_backward");
    set(api.short_conv_step, "vsv_short_conv_step");
    set(api.ssm_saved_floats, "vsv_ssm_saved_floats");
    set(api.ssm_scan_ws_bytes, "vsv_ssm_scan_ws_bytes");
    set(api.ssm_scan, "vsv_ssm_scan");
    set(api.ssm_scan_backward_ws_bytes, "vsv_ssm_scan_backward_ws_bytes");
    set(api.ssm_scan_backward, "vsv_ssm_scan_backward");
    set(api.ssm_step, "vsv_ssm_step");
    set(api.adamw_multi, "vsv_adamw_multi");
    set(api.adamw_read8, "vsv_adamw_read8");
    set(api.last_error, "vsv_last_error");
}

// As vsv/lib.py's check: a negative code is an argument's fault, a positive one a HIP error.
void check(int rc, const char* what) {
    TORCH_CHECK_VALUE(rc >= 0, what, ": ", api.last_error());
    TORCH_CHECK(rc == 0, what, ": HIP error ", rc, ": ", api.last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return VSV_F32;
        case at::kBFloat16: return VSV_BF16;
        case at::kHalf: return VSV_F16;
        default: return -1;
    }
}

Tensor last_contiguous(const Tensor& t_) {
    const Tensor t = t_.resolve_neg();                                     // (a conjugate's imaginary part is a view with its sign put off)
    if (t.is_contiguous()) return t;
    return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

Tensor seq(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape, std::optional<at::ScalarType> type) {
    TORCH_CHECK_VALUE(t.sizes() == shape, what, ": ", name, " must be a tensor of shape ", shape, ", not ", t.sizes());
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && type_code(t) >= 0, what, ": ", name, " must be float32, bfloat16 or float16, not ", t.scalar_type());
    TORCH_CHECK_VALUE(!type || t.scalar_type() == *type, what, ": ", name, " must be ", *type, " as x is, not ", t.scalar_type());
    return last_contiguous(t);
}

Tensor f32(const char* what, const char* name, const OptTensor& t, at::IntArrayRef shape) {
    if (!t || !t->defined()) return Tensor();
    TORCH_CHECK_VALUE(t->sizes() == shape && t->scalar_type() == at::kFloat && t->layout() == at::kStrided, what, ": ", name,
                      " must be a float32 tensor of shape ", shape, ", not ", t->scalar_type(), " ", t->sizes());
    return t->resolve_neg().contiguous();
}

Tensor int_lengths(const char* what, const OptTensor& t, int64_t B) {
    if (!t || !t->defined()) return Tensor();
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == B && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong), what,
                      ": lengths must be an int32 or int64 tensor of shape [", B, "]");
    if (t->scalar_type() == at::kLong) return t->clamp(0, 0x7fffffff).to(at::kInt).contiguous();
    return t->contiguous();
}

void in_place(const char* what, const Tensor& t, at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(t.sizes() == shape && t.scalar_type() == at::kFloat && t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg(), what,
                      ": state must be a contiguous float32 tensor of shape ", shape, " (it is updated in place)");
}

void same_gpu(const char* what, const Tensor& x, std::initializer_list<Tensor> others) {
    TORCH_CHECK(x.is_cuda(), what, ": tensors must be on a GPU; there is no CPU fallback");
    for (const Tensor& t : others)
        TORCH_CHECK_VALUE(!t.defined() || t.device() == x.device(), what, ": tensors are on ", t.device(), " and ", x.device());
}

bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// A tangent would be dropped without a word: what follows looks at requires_grad and at memory alone.  (No level, no tangents:
// the usual call asks once, as a question to every tensor took the host 0.5 us a call.)
template <typename... Ts> void no_tangents(const char* what, const Ts&... ts) {
    if (!torch::autograd::ForwardADLevel::try_get_by_idx(0)) return;
    auto one = [&](const Tensor& t) {
        TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward-mode derivative, and an input carries a tangent");
    };
    (one(ts), ...);
}

// A tracer sees none of the calls below: it would keep this call's outputs as constants.
void not_traced(const char* what) { TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced"); }

Tensor given(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
// (straight from the allocator: through the dispatcher a tensor costs the host twice as much, and a backward pass makes twelve)
Tensor fresh(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) { return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt)); }
Tensor whole_like(const Tensor& t) { return fresh(t, t.sizes(), t.scalar_type()); }
Tensor floats(const Tensor& like, at::IntArrayRef shape) { return fresh(like, shape, at::kFloat); }
Tensor workspace(const Tensor& like, size_t bytes) { return fresh(like, {(int64_t)(bytes ? bytes : 16)}, at::kByte); }
// what a backward pass returns for an input: nothing where no gradient was asked for
Tensor grad_like(const Tensor& input) { return input.defined() && input.requires_grad() ? whole_like(input) : Tensor(); }
Tensor asked(const Tensor& input, const Tensor& grad) { return input.defined() && input.requires_grad() ? grad : Tensor(); }

template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }

// With create_graph the gradients carry an error for whoever differentiates them again.
variable_list once(variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list defined;
    for (const Tensor& g : grads)
        if (g.defined()) defined.push_back(g.detach().requires_grad_(true));
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative", (int64_t)defined.size());
    variable_list marked = (*node)(std::move(defined));
    size_t k = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = marked[k++];
    return grads;
}

// ---- short causal convolution ------------------------------------------------------------------------------------

vsv_short_conv_desc conv_desc(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& h0, const Tensor& lengths, bool silu, void* y,
                              const Tensor& state) {
    vsv_short_conv_desc d = {};
    d.dtype = type_code(x); d.K = (int)w.size(1); d.silu = silu;
    d.B = x.size(0); d.T = x.dim() == 3 ? x.size(1) : 1; d.D = x.size(-1);
    d.x = x.data_ptr(); d.x_bs = x.stride(0); d.x_ts = x.dim() == 3 ? x.stride(1) : 0;
    d.w = ptr<float>(w); d.bias = ptr<float>(bias); d.state_in = ptr<float>(h0); d.lengths = ptr<int>(lengths);
    d.y = y; d.state_out = ptr<float>(state);
    return d;
}

variable_list conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& h0, const Tensor& lengths, bool silu, bool want) {
    c10::DeviceGuard guard(x.device());
    Tensor y = whole_like(x), state = want ? floats(x, {x.size(0), w.size(1) - 1, x.size(2)}) : Tensor();
    const auto d = conv_desc(x, w, bias, h0, lengths, silu, y.data_ptr(), state);
    check(api.short_conv(&d, stream_of(x)), "vsv_short_conv");
    if (want) return {y, state};
    return {y};
}

struct ShortConv : torch::autograd::Function<ShortConv> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_, const OptTensor& h0_,
                                 const OptTensor& lengths_, bool silu, bool want) {
        const Tensor bias = given(bias_), h0 = given(h0_), lengths = given(lengths_);
        ctx->save_for_backward({x, w, bias, h0, lengths});
        ctx->saved_data["silu"] = silu;
        ctx->set_materialize_grads(false);
        return conv_forward(x, w, bias, h0, lengths, silu, want);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &bias = saved[2], &h0 = saved[3], &lengths = saved[4];
        Tensor dy = grads[0], dstate = grads.size() > 1 ? grads[1] : Tensor();
        if (!dy.defined() && !dstate.defined()) return variable_list(7);
        no_tangents("short_conv's backward pass", dy, dstate);
        Tensor dx, dw, db, dh;
        {
            at::NoGradGuard no_grad;
            c10::DeviceGuard guard(x.device());
            dy = dy.defined() ? last_contiguous(dy) : at::zeros_like(x, x.options(), at::MemoryFormat::Contiguous);
            if (dstate.defined()) dstate = dstate.resolve_neg().contiguous();
            dx = whole_like(x);
            dw = grad_like(w);
            db = grad_like(bias);
            dh = grad_like(h0);
            const auto d = conv_desc(x, w, bias, h0, lengths, ctx->saved_data["silu"].toBool(), dx.data_ptr(), Tensor());
            vsv_short_conv_grads g = {};
            g.dy = dy.data_ptr(); g.dy_bs = dy.stride(0); g.dy_ts = dy.stride(1); g.d_state_out = ptr<float>(dstate);
            g.dx = dx.data_ptr(); g.dw = ptr<float>(dw); g.dbias = ptr<float>(db); g.d_state_in = ptr<float>(dh);
            const size_t bytes = api.short_conv_backward_ws_bytes(&d);
            const Tensor ws = workspace(x, bytes);
            check(api.short_conv_backward(&d, &g, ws.data_ptr(), bytes, stream_of(x)), "vsv_short_conv_backward");
        }
        return once({asked(x, dx), dw, db, dh, Tensor(), Tensor(), Tensor()}, "short_conv");
    }
};

void conv_weight(const char* what, const Tensor& x, const Tensor& weight) {
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) >= 1 && weight.size(1) <= VSV_CONV_MAX_TAPS && x.size(-1) >= 1, what,
                      ": weight must be a tensor (D, K) with 1 to ", VSV_CONV_MAX_TAPS, " taps");
}

variable_list short_conv(const Tensor& x_, const Tensor& weight, const OptTensor& bias_, bool silu, const OptTensor& state_, const OptTensor& lengths_,
                         bool want) {
    const char* what = "short_conv";
    TORCH_CHECK_VALUE(x_.dim() == 3, what, ": x must be a tensor (B, T, D)");
    conv_weight(what, x_, weight);
    const int64_t B = x_.size(0), D = x_.size(2), K = weight.size(1);
    const Tensor x = seq(what, "x", x_, x_.sizes(), std::nullopt);
    const Tensor w = f32(what, "weight", weight, {D, K}), bias = f32(what, "bias", bias_, {D}), h0 = f32(what, "initial_state", state_, {B, K - 1, D});
    const Tensor lengths = int_lengths(what, lengths_, B);
    not_traced(what);
    no_tangents(what, x, w, bias, h0);
    same_gpu(what, x, {w, bias, h0, lengths});
    if (wants_grad({x, w, bias, h0})) return ShortConv::apply(x, w, opt(bias), opt(h0), opt(lengths), silu, want);
    return conv_forward(x, w, bias, h0, lengths, silu, want);
}

Tensor short_conv_step(const Tensor& x_, const Tensor& state, const Tensor& weight, const OptTensor& bias_, bool silu) {
    const char* what = "short_conv_step";
    TORCH_CHECK_VALUE(x_.dim() == 2, what, ": x must be a tensor (B, D)");
    conv_weight(what, x_, weight);
    const int64_t B = x_.size(0), D = x_.size(1), K = weight.size(1);
    const Tensor x = seq(what, "x", x_, x_.sizes(), std::nullopt), w = f32(what, "weight", weight, {D, K}), bias = f32(what, "bias", bias_, {D});
    in_place(what, state, {B, K - 1, D});
    not_traced(what);
    no_tangents(what, x, w, bias, state);
    same_gpu(what, x, {w, bias, state});
    TORCH_CHECK(!wants_grad({x, w, bias, state}), what, " has no gradient: call it under torch.no_grad()");
    c10::DeviceGuard guard(x.device());
    const Tensor y = whole_like(x);
    const auto d = conv_desc(x, w, bias, Tensor(), Tensor(), silu, y.data_ptr(), state);
    state.unsafeGetTensorImpl()->bump_version();                           // (refuses an inference tensor outside inference mode)
    check(api.short_conv_step(&d, stream_of(x)), "vsv_short_conv_step");
    return y;
}

// ---- selective scan ----------------------------------------------------------------------------------------------

struct ScanArgs { Tensor x, dt, a, b, c, skip, gate, dt_bias; };

Tensor grouped(const char* what, const char* name, const Tensor& t_, at::IntArrayRef lead, int64_t D, int64_t N, at::ScalarType type) {
    const int64_t dims = (int64_t)lead.size();
    const Tensor t = t_.dim() == dims + 1 ? t_.unsqueeze(-2) : t_;
    TORCH_CHECK_VALUE(t.dim() == dims + 2 && t.size(-2) >= 1 && D % t.size(-2) == 0, what, ": ", name, " must be a tensor (..., [G,] N) over ", lead,
                      " with G a divisor of D = ", D);
    c10::SmallVector<int64_t, 4> shape(lead.begin(), lead.end());
    shape.push_back(t.size(-2));
    shape.push_back(N);
    return seq(what, name, t, shape, type);
}

ScanArgs scan_args(const char* what, const Tensor& x_, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& skip,
                   const OptTensor& gate, const OptTensor& dt_bias) {
    const int64_t D = x_.size(-1);
    TORCH_CHECK_VALUE(a.dim() == 2 && a.size(0) == D && a.size(1) >= 1 && a.size(1) <= VSV_SSM_MAX_STATE && D >= 1, what,
                      ": a must be a tensor (D, N) with 1 to ", VSV_SSM_MAX_STATE, " states");
    const int64_t N = a.size(1);
    ScanArgs r;
    r.x = seq(what, "x", x_, x_.sizes(), std::nullopt);
    const auto type = r.x.scalar_type();
    r.dt = seq(what, "dt", dt, x_.sizes(), type);
    if (gate && gate->defined()) r.gate = seq(what, "gate", *gate, x_.sizes(), type);
    const auto lead = x_.sizes().slice(0, x_.dim() - 1);
    r.b = grouped(what, "b", b, lead, D, N, type);
    r.c = grouped(what, "c", c, lead, D, N, type);
    TORCH_CHECK_VALUE(r.b.size(-2) == r.c.size(-2), what, ": b has ", r.b.size(-2), " groups and c ", r.c.size(-2));
    r.a = f32(what, "a", a, {D, N});
    r.skip = f32(what, "skip", skip, {D});
    r.dt_bias = f32(what, "dt_bias", dt_bias, {D});
    return r;
}

vsv_ssm_desc scan_desc(const ScanArgs& r, const Tensor& h0, const Tensor& lengths, bool softplus, void* y, const Tensor& state) {
    vsv_ssm_desc d = {};
    const bool time = r.x.dim() == 3;
    auto ts = [&](const Tensor& t) { return time ? t.stride(1) : 0; };
    d.dtype = type_code(r.x); d.N = (int)r.a.size(1); d.softplus = softplus;
    d.B = r.x.size(0); d.T = time ? r.x.size(1) : 1; d.D = r.x.size(-1); d.G = r.b.size(-2);
    d.x = r.x.data_ptr(); d.x_bs = r.x.stride(0); d.x_ts = ts(r.x);
    d.dt = r.dt.data_ptr(); d.dt_bs = r.dt.stride(0); d.dt_ts = ts(r.dt);
    if (r.gate.defined()) { d.gate = r.gate.data_ptr(); d.gate_bs = r.gate.stride(0); d.gate_ts = ts(r.gate); }
    d.b = r.b.data_ptr(); d.b_bs = r.b.stride(0); d.b_ts = ts(r.b); d.b_gs = r.b.stride(-2);
    d.c = r.c.data_ptr(); d.c_bs = r.c.stride(0); d.c_ts = ts(r.c); d.c_gs = r.c.stride(-2);
    d.a = ptr<float>(r.a); d.skip = ptr<float>(r.skip); d.dt_bias = ptr<float>(r.dt_bias);
    d.state_in = ptr<float>(h0); d.lengths = ptr<int>(lengths); d.y = y; d.state_out = ptr<float>(state);
    return d;
}

variable_list scan_forward(const ScanArgs& r, const Tensor& h0, const Tensor& lengths, bool softplus, bool want, Tensor* saved) {
    c10::DeviceGuard guard(r.x.device());
    Tensor y = whole_like(r.x), state = want ? floats(r.x, {r.x.size(0), r.x.size(2), r.a.size(1)}) : Tensor();
    auto d = scan_desc(r, h0, lengths, softplus, y.data_ptr(), state);
    if (saved) {
        *saved = floats(r.x, {(int64_t)api.ssm_saved_floats(&d)});
        d.saved = ptr<float>(*saved);
    }
    const size_t bytes = api.ssm_scan_ws_bytes(&d);
    const Tensor ws = bytes ? workspace(r.x, bytes) : Tensor();
    check(api.ssm_scan(&d, ptr(ws), bytes, stream_of(r.x)), "vsv_ssm_scan");
    if (want) return {y, state};
    return {y};
}

struct SsmScan : torch::autograd::Function<SsmScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c,
                                 const OptTensor& skip_, const OptTensor& gate_, const OptTensor& dt_bias_, const OptTensor& h0_,
                                 const OptTensor& lengths_, bool softplus, bool want) {
        const Tensor skip = given(skip_), gate = given(gate_), dt_bias = given(dt_bias_), h0 = given(h0_), lengths = given(lengths_);
        Tensor saved;
        variable_list out = scan_forward({x, dt, a, b, c, skip, gate, dt_bias}, h0, lengths, softplus, want, &saved);
        ctx->save_for_backward({x, dt, a, b, c, skip, gate, dt_bias, h0, lengths, saved});
        ctx->saved_data["softplus"] = softplus;
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const ScanArgs r = {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]};
        const Tensor &h0 = s[8], &lengths = s[9], &saved = s[10];
        Tensor dy = grads[0], dstate = grads.size() > 1 ? grads[1] : Tensor();
        if (!dy.defined() && !dstate.defined()) return variable_list(12);
        no_tangents("ssm_scan's backward pass", dy, dstate);
        Tensor dx, ddt, dgate, db, dc, da, dskip, dbias, dh;
        {
            at::NoGradGuard no_grad;
            c10::DeviceGuard guard(r.x.device());
            dy = dy.defined() ? last_contiguous(dy) : at::zeros_like(r.x, r.x.options(), at::MemoryFormat::Contiguous);
            if (dstate.defined()) dstate = dstate.resolve_neg().contiguous();
            dx = whole_like(r.x); ddt = whole_like(r.x); db = whole_like(r.b); dc = whole_like(r.c);
            if (r.gate.defined()) dgate = whole_like(r.x);
            da = grad_like(r.a); dskip = grad_like(r.skip); dbias = grad_like(r.dt_bias); dh = grad_like(h0);
            auto d = scan_desc(r, h0, lengths, ctx->saved_data["softplus"].toBool(), dx.data_ptr(), Tensor());
            d.saved = ptr<float>(saved);
            vsv_ssm_grads g = {};
            g.dy = dy.data_ptr(); g.dy_bs = dy.stride(0); g.dy_ts = dy.stride(1); g.d_state_out = ptr<float>(dstate);
            g.dx = dx.data_ptr(); g.ddt = ddt.data_ptr(); g.dgate = ptr(dgate); g.db = db.data_ptr(); g.dc = dc.data_ptr();
            g.da = ptr<float>(da); g.dskip = ptr<float>(dskip); g.ddt_bias = ptr<float>(dbias); g.d_state_in = ptr<float>(dh);
            const size_t bytes = api.ssm_scan_backward_ws_bytes(&d);
            const Tensor ws = workspace(r.x, bytes);
            check(api.ssm_scan_backward(&d, &g, ws.data_ptr(), bytes, stream_of(r.x)), "vsv_ssm_scan_backward");
        }
        return once({asked(r.x, dx), asked(r.dt, ddt), da, asked(r.b, db), asked(r.c, dc), dskip, asked(r.gate, dgate), dbias, dh, Tensor(), Tensor(),
                     Tensor()}, "ssm_scan");
    }
};

variable_list ssm_scan(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& skip,
                       const OptTensor& gate, const OptTensor& dt_bias, bool softplus, const OptTensor& state_, const OptTensor& lengths_, bool want) {
    const char* what = "ssm_scan";
    TORCH_CHECK_VALUE(x.dim() == 3, what, ": x must be a tensor (B, T, D)");
    const ScanArgs r = scan_args(what, x, dt, a, b, c, skip, gate, dt_bias);
    const Tensor h0 = f32(what, "initial_state", state_, {x.size(0), x.size(2), a.size(1)}), lengths = int_lengths(what, lengths_, x.size(0));
    not_traced(what);
    no_tangents(what, r.x, r.dt, r.a, r.b, r.c, r.skip, r.gate, r.dt_bias, h0);
    same_gpu(what, r.x, {r.dt, r.a, r.b, r.c, r.skip, r.gate, r.dt_bias, h0, lengths});
    if (wants_grad({r.x, r.dt, r.a, r.b, r.c, r.skip, r.gate, r.dt_bias, h0}))
        return SsmScan::apply(r.x, r.dt, r.a, r.b, r.c, opt(r.skip), opt(r.gate), opt(r.dt_bias), opt(h0), opt(lengths), softplus, want);
    return scan_forward(r, h0, lengths, softplus, want, nullptr);
}

Tensor ssm_step(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& skip, const OptTensor& gate,
                const Tensor& state, const OptTensor& dt_bias, bool softplus) {
    const char* what = "ssm_step";
    TORCH_CHECK_VALUE(x.dim() == 2, what, ": x must be a tensor (B, D)");
    const ScanArgs r = scan_args(what, x, dt, a, b, c, skip, gate, dt_bias);
    in_place(what, state, {x.size(0), x.size(1), a.size(1)});
    not_traced(what);
    no_tangents(what, r.x, r.dt, r.a, r.b, r.c, r.skip, r.gate, r.dt_bias, state);
    same_gpu(what, r.x, {r.dt, r.a, r.b, r.c, r.skip, r.gate, r.dt_bias, state});
    TORCH_CHECK(!wants_grad({r.x, r.dt, r.a, r.b, r.c, r.skip, r.gate, r.dt_bias, state}), what, " has no gradient: call it under torch.no_grad()");
    c10::DeviceGuard guard(r.x.device());
    const Tensor y = whole_like(r.x);
    const auto d = scan_desc(r, Tensor(), Tensor(), softplus, y.data_ptr(), state);
    state.unsafeGetTensorImpl()->bump_version();
    check(api.ssm_step(&d, stream_of(r.x)), "vsv_ssm_step");
    return y;
}

// ---- AdamW -------------------------------------------------------------------------------------------------------

using Tensors = std::vector<Tensor>;
// parameters, gradients, exp_avg, exp_avg_sq, their scales (8 bits); lr, beta1, beta2, eps, weight_decay; the step's number
using AdamwCall = std::tuple<Tensors, Tensors, Tensors, Tensors, Tensors, Tensors, double, double, double, double, double, int64_t>;

void state_fits(const Tensor& p, const Tensor& t, at::ScalarType type, int64_t n) {
    TORCH_CHECK_VALUE(t.numel() == n && t.scalar_type() == type && t.device() == p.device() && t.is_contiguous() && !t.is_neg(),
                      "AdamW: a parameter has changed its shape or device since its state was made");
}

// One launch updates the tensors side by side, so none may hold another's elements.
void apart(std::vector<std::pair<uintptr_t, uintptr_t>>& spans) {
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK_VALUE(spans[i - 1].second <= spans[i].first, "AdamW: two parameters share memory");
}

void refuse_capture() {                                                    // of the current device's current stream
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None,
                "AdamW.step cannot be captured into a HIP graph: the step count is a launch argument");
}

void adamw_step(int bits, std::vector<AdamwCall> calls) {
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (auto& [p, g, m, v, ms, vs, lr, b1, b2, eps, wd, step] : calls) {   // everything is checked before anything is launched
        TORCH_CHECK_VALUE(lr >= 0.0 && b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && eps >= 0.0 && wd >= 0.0, "AdamW: bad hyper-parameters lr=", lr,
                          " betas=(", b1, ", ", b2, ") eps=", eps, " weight_decay=", wd);
        for (size_t i = 0; i < p.size(); ++i) {
            TORCH_CHECK_VALUE(type_code(p[i]) >= 0, "AdamW: parameters must be float32, bfloat16 or float16, not ", p[i].scalar_type());
            TORCH_CHECK_VALUE(p[i].is_contiguous() && !p[i].is_neg(), "AdamW: parameters must be contiguous, and no negative views");
            TORCH_CHECK_VALUE(g[i].layout() == at::kStrided && g[i].scalar_type() == p[i].scalar_type() && g[i].device() == p[i].device() &&
                                  g[i].sizes() == p[i].sizes(), "AdamW: a gradient needs its parameter's type, device and shape, and no sparse layout");
            const uintptr_t at = (uintptr_t)p[i].data_ptr();
            if (p[i].numel()) spans.push_back({at, at + p[i].nbytes()});
            const int64_t n = p[i].numel(), blocks = (n + VSV_ADAMW_BLOCK - 1) / VSV_ADAMW_BLOCK;
            state_fits(p[i], m[i], bits == 8 ? at::kChar : at::kFloat, n);
            state_fits(p[i], v[i], bits == 8 ? at::kByte : at::kFloat, n);
            if (bits == 8) { state_fits(p[i], ms[i], at::kFloat, blocks); state_fits(p[i], vs[i], at::kFloat, blocks); }
        }
    }
    apart(spans);
    at::Device asked(at::kCPU);
    for (const auto& call : calls)
        for (const Tensor& p : std::get<0>(call)) {
            if (!p.is_cuda() || p.device() == asked) continue;
            asked = p.device();
            c10::DeviceGuard guard(asked);
            refuse_capture();
        }
    for (auto& call : calls) {
        auto& [p, g, m, v, ms, vs, lr, b1, b2, eps, wd, step] = call;
        for (size_t i = 0; i < p.size(); ++i) {
            TORCH_CHECK(p[i].is_cuda(), "AdamW: parameters must be on a GPU; there is no CPU fallback");
            for (const Tensor& t : {p[i], m[i], v[i]}) t.unsafeGetTensorImpl()->bump_version();
            g[i] = g[i].resolve_neg().contiguous();
        }
    }
    for (auto& [p, g, m, v, ms, vs, lr, b1, b2, eps, wd, step] : calls) {
        std::vector<char> done(p.size(), 0);
        for (size_t first = 0; first < p.size(); ++first) {                 // one call per type and device
            if (done[first]) continue;
            std::vector<vsv_adamw_tensor> table;
            for (size_t i = first; i < p.size(); ++i) {
                if (done[i] || p[i].scalar_type() != p[first].scalar_type() || p[i].device() != p[first].device()) continue;
                done[i] = 1;
                table.push_back({p[i].data_ptr(), g[i].data_ptr(), m[i].data_ptr(), v[i].data_ptr(), bits == 8 ? ptr<float>(ms[i]) : nullptr,
                                 bits == 8 ? ptr<float>(vs[i]) : nullptr, (long)p[i].numel()});
            }
            c10::DeviceGuard guard(p[first].device());
            check(api.adamw_multi(table.data(), (int)table.size(), type_code(p[first]), bits, lr, b1, b2, eps, wd, step, stream_of(p[first])),
                  "vsv_adamw_multi");
        }
    }
}

std::pair<Tensors, Tensors> adamw_read8(const Tensors& m, const Tensors& v, const Tensors& ms, const Tensors& vs) {
    Tensors mo, vo;
    for (const Tensor& t : m) {
        mo.push_back(floats(t, t.sizes()));
        vo.push_back(floats(t, t.sizes()));
    }
    std::vector<char> done(m.size(), 0);
    for (size_t first = 0; first < m.size(); ++first) {
        if (done[first]) continue;
        std::vector<vsv_adamw_tensor> table;
        for (size_t i = first; i < m.size(); ++i) {
            if (done[i] || m[i].device() != m[first].device()) continue;
            done[i] = 1;
            table.push_back({mo[i].data_ptr(), vo[i].data_ptr(), m[i].data_ptr(), v[i].data_ptr(), ptr<float>(ms[i]), ptr<float>(vs[i]), (long)m[i].numel()});
        }
        c10::DeviceGuard guard(m[first].device());
        check(api.adamw_read8(table.data(), (int)table.size(), stream_of(m[first])), "vsv_adamw_read8");
    }
    return {mo, vo};
}

}  // namespace

PYBIND11_MODULE(_vsv_torch, m) {
    m.def("bind", &bind);
    m.def("short_conv", &short_conv);
    m.def("short_conv_step", &short_conv_step);
    m.def("ssm_scan", &ssm_scan);
    m.def("ssm_step", &ssm_step);
    m.def("adamw_step", &adamw_step);
    m.def("refuse_capture", &refuse_capture);
    m.def("adamw_read8", &adamw_read8);
}
