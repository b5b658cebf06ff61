// The operators around the attention call as torch functions: allocation, description and launch, and the autograd nodes.
//
// These calls are short (a backward pass of a small layer keeps the GPU busy for 20 us), and a training step makes dozens
// of them, so what the host does per call counts: the same binding written in Python took 15 us forward and, on
// autograd's own thread with its interpreter lock handed back and forth, 46 us backward.  Nothing here computes: every
// function checks sizes, allocates outputs and workspace as tensors, fills one plain struct of include/fwa2.h and calls
// the library on the current stream of the tensors' device.  The arguments' types and shapes are checked by the
// Python functions in block_ops.py that call this.
#include <torch/extension.h>

#include <ATen/FuncTorchTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/fwa2.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Optional;

// A status of the library, on its way to the exception that _abi.check raises for it.
struct StatusError : std::runtime_error {
    int code;
    StatusError(int c, const std::string& what) : std::runtime_error(what), code(c) {}
};
void check(int status, const char* what) {
    if (status == FWA2_OK) return;
    throw StatusError(status, std::string(what) + ": " + fwa2_last_error());
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return FWA2_F16;
        case at::kBFloat16: return FWA2_BF16;
        case at::kFloat: return FWA2_F32;
        case at::kFloat8_e4m3fn: return FWA2_E4M3;
        default: throw StatusError(FWA2_ERR_INVALID_ARGUMENT, "unsupported dtype");
    }
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor value(const Optional& t) { return t.has_value() ? *t : Tensor(); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor make(at::IntArrayRef shape, const Tensor& like, at::ScalarType t) { return at::empty(shape, like.options().dtype(t).requires_grad(false)); }

int64_t row_count(const Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i + 1 < t.dim(); i++) n *= t.size(i);
    return n;
}

// The tensor itself, unless it is a view that negates what its memory holds (the imaginary part of a conjugate is one).
Tensor as_held(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return as_held(t).contiguous(); }

// A tensor as [rows, last] with unit inner stride: itself where the kernels can address it, a copy otherwise (inner stride
// other than 1, rows that overlap or lie 2^22 elements apart or more).  The tensor lives as long as this does.
struct Rows {
    Tensor t;
    void* ptr = nullptr;
    int64_t stride = 0;
    Rows() = default;
    explicit Rows(const Tensor& from) : t(as_held(from)) {
        const int64_t last = t.size(-1);
        stride = last;
        if (!t.is_contiguous()) {
            t = t.reshape({-1, last});
            const bool inner = last == 1 || t.stride(1) == 1;
            if (t.size(0) <= 1) {
                if (!inner) t = t.contiguous();
            } else {
                if (!inner || t.stride(0) < last || t.stride(0) >= (1 << 22)) t = t.contiguous();
                stride = t.stride(0);
            }
        }
        ptr = t.data_ptr();
    }
};

// Gradients computed here have no graph of their own: in a backward pass that records one, differentiating them again has
// to fail instead of giving zeros.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads) {
        if (!g.defined()) continue;
        variable_list one = {g.detach().requires_grad_(true)};
        auto fn = std::make_shared<torch::autograd::DelayedError>("the operator's gradient cannot be differentiated a second time", 1);
        g = (*fn)(std::move(one))[0];
    }
    return grads;
}

bool wants_grad(std::initializer_list<const Optional*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Optional* t : ts)
        if (t->has_value() && (*t)->defined() && (*t)->requires_grad()) return true;
    return false;
}

// What follows a computation from outside does not see into these functions.  A backward pass is recorded by their nodes; a
// forward-mode derivative that an input carries would be lost, and so would what the transforms of torch.func keep; a tracer
// would record that an output is allocated and not what fills it.
bool has_forward_grad(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_forward_grad(const Optional& t) { return t.has_value() && has_forward_grad(*t); }
template <class... T>
void refuse_unseen(const T&... ts) {
    if ((has_forward_grad(ts) || ...)) throw StatusError(FWA2_ERR_UNSUPPORTED, "the operator has no forward-mode derivative");
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
        throw StatusError(FWA2_ERR_UNSUPPORTED, "the operator cannot be traced");
    if (const auto& transforms = at::functorch::functorchTLSAccessor()) transforms->checkSupportsCppAutogradFunction();
}

// ---- matrix products ----
fwa2_linear linear_description(const Rows& x, const Rows& w, int64_t rows, int64_t k, int64_t n, at::ScalarType t, at::ScalarType xt, int act) {
    fwa2_linear p = {};
    p.struct_bytes = sizeof(p);
    p.abi_version = FWA2_ABI_VERSION;
    p.dtype = dtype_code(t);
    p.x_dtype = dtype_code(xt);
    p.activation = act;
    TORCH_CHECK(k <= INT32_MAX && n <= INT32_MAX, "fused linear: a matrix extent is beyond 2^31");
    p.in_features = (int)k;
    p.out_features = (int)n;
    p.rows = rows;
    p.x = x.ptr; p.x_stride = x.stride;
    p.weight = w.ptr; p.weight_stride = w.stride;
    return p;
}
void linear_run(fwa2_linear& p, const Tensor& like, bool backward) {
    Tensor ws;
    if (const size_t need = fwa2_linear_workspace_bytes(&p, backward)) {
        ws = make({(int64_t)need}, like, at::kByte);
        p.workspace = ws.data_ptr();
        p.workspace_bytes = need;
    }
    p.stream = stream_of(like);
    if (backward) check(fwa2_linear_backward(&p), "fwa2_linear_backward");
    else check(fwa2_linear_forward(&p), "fwa2_linear_forward");
}

// (y, z): z, the sums before the activation, only if asked for
std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight, const Optional& bias, int act, const Optional& residual,
                                         at::ScalarType t, bool want_z, const Optional& x_scale, const Optional& w_scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = row_count(x), k = weight.size(1), n = weight.size(0);
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    Tensor y = make(shape, x, t), z;
    if (want_z) z = make(shape, x, t);
    if (rows == 0) return {y, z};
    const Rows xr(x), wr(weight);
    Rows rr;
    fwa2_linear p = linear_description(xr, wr, rows, k, n, t, x.scalar_type(), act);
    Tensor b, xs, ws;
    if (bias) { b = dense(*bias); p.bias = b.data_ptr(); }
    if (residual) { rr = Rows(*residual); p.residual = rr.ptr; p.residual_stride = rr.stride; }
    if (x_scale) {
        xs = dense(*x_scale); ws = dense(*w_scale);
        p.x_scale = xs.data_ptr<float>(); p.weight_scale = ws.data_ptr<float>();
    }
    p.y = ptr(y); p.z = ptr(z);
    linear_run(p, x, false);
    return {y, z};
}

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Optional& bias, const Optional& residual, int64_t act,
                          bool want_z) {
        auto [y, z] = linear_forward(x, weight, bias, (int)act, residual, x.scalar_type(), want_z, std::nullopt, std::nullopt);
        ctx->save_for_backward({x, weight, z});
        ctx->saved_data["how"] = act * 4 + (bias ? 1 : 0) + (residual ? 2 : 0);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &z = saved[2], &dy = grads[0];
        refuse_unseen(dy);
        const int64_t how = ctx->saved_data["how"].toInt();
        const bool has_bias = how & 1, has_residual = how & 2;
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_bias && ctx->needs_input_grad(2),
                   need_r = has_residual && ctx->needs_input_grad(2 + has_bias);
        Tensor dx, dw, db;
        if (dy.defined()) {
            at::AutoDispatchBelowADInplaceOrView below;
            const c10::DeviceGuard guard(x.device());
            const int64_t rows = row_count(x);
            if (need_x) dx = make(x.sizes(), x, x.scalar_type());
            if (need_w || need_b) dw = make(weight.sizes(), x, x.scalar_type());    // dbias is summed on the way to dweight
            if (need_b) db = make({weight.size(0)}, x, x.scalar_type());
            if (rows == 0) {
                if (dw.defined()) dw.zero_();
                if (db.defined()) db.zero_();
            } else if (dx.defined() || dw.defined()) {
                const Rows xr(x), wr(weight), dyr(dy);
                fwa2_linear p = linear_description(xr, wr, rows, weight.size(1), weight.size(0), x.scalar_type(), x.scalar_type(), (int)(how / 4));
                p.dy = dyr.ptr; p.dy_stride = dyr.stride;
                p.z = ptr(z); p.dx = ptr(dx); p.dweight = ptr(dw); p.dbias = ptr(db);
                linear_run(p, x, true);
            }
        }
        return once({dx, need_w ? dw : Tensor(), db, need_r ? dy : Tensor(), Tensor(), Tensor()});
    }
};

Tensor linear(const Tensor& x, const Tensor& weight, const Optional& bias, int64_t act, const Optional& residual) {
    refuse_unseen(x, weight, bias, residual);
    const Optional xo(x), wo(weight);
    if (wants_grad({&xo, &wo, &bias, &residual}))
        return LinearNode::apply(x, weight, bias, residual, act, act != FWA2_ACT_NONE && wants_grad({&xo, &wo, &bias}));
    return linear_forward(x, weight, bias, (int)act, residual, x.scalar_type(), false, std::nullopt, std::nullopt).first;
}

Tensor linear_fp8(const Tensor& x8, const Tensor& x_scale, const Tensor& weight8, const Tensor& weight_scale, const Optional& bias, int64_t act,
                  const Optional& residual, bool bf16) {
    refuse_unseen(x_scale, weight_scale, bias, residual);
    return linear_forward(x8, weight8, bias, (int)act, residual, bf16 ? at::kBFloat16 : at::kHalf, false, x_scale, weight_scale).first;
}

// ---- normalisation ----
struct NormHow {
    double eps;
    int kind, place;
    at::ScalarType x, stream;
    bool pre() const { return place == FWA2_NORM_PRE; }
    bool exact_h() const { return pre() && stream == at::kFloat; }
    bool two() const { return pre() && stream != at::kFloat; }
};
struct NormParams {     // weight, bias and gate, contiguous, for as long as the call needs them
    Tensor weight, bias, gate;
};

fwa2_norm norm_description(const Tensor& v, const NormHow& how, const Tensor& weight, const Tensor& bias, const Tensor& gate, NormParams& keep) {
    fwa2_norm p = {};
    p.struct_bytes = sizeof(p);
    p.abi_version = FWA2_ABI_VERSION;
    p.dtype = dtype_code(how.x); p.stream_dtype = dtype_code(how.stream); p.param_dtype = dtype_code(weight.scalar_type());
    p.kind = how.kind; p.placement = how.place; p.eps = (float)how.eps;
    p.rows = row_count(v);
    TORCH_CHECK(v.size(-1) <= INT32_MAX, "norm: rows of more than 2^31 values");
    p.dim = (int)v.size(-1);
    keep.weight = dense(weight);
    p.weight = keep.weight.data_ptr();
    if (bias.defined()) { keep.bias = dense(bias); p.bias = keep.bias.data_ptr(); }
    if (gate.defined()) {
        keep.gate = dense(gate);
        p.gate = keep.gate.data_ptr();
        p.gate_dtype = dtype_code(gate.scalar_type());
        p.rows_per_gate = p.rows / gate.numel();
    }
    return p;
}

struct NormOut {
    Tensor y, h, y8, scale, stats;
};
NormOut norm_forward(const Tensor& x, const Optional& shortcut, const Tensor& weight, const Optional& bias, const Optional& gate,
                     const NormHow& how, bool want_stats, bool want_y8) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = row_count(x);
    NormOut o;
    if (how.pre()) o.h = make(x.sizes(), x, how.stream);
    if (!how.pre() || !want_y8) o.y = make(x.sizes(), x, how.pre() ? how.x : how.stream);
    if (want_y8) {
        o.y8 = make(x.sizes(), x, at::kFloat8_e4m3fn);
        o.scale = make(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
    }
    if (want_stats) o.stats = make({rows, 2}, x, at::kFloat);
    if (rows == 0) return o;
    NormParams keep;
    fwa2_norm p = norm_description(x, how, weight, value(bias), value(gate), keep);
    const Rows xr(x);
    Rows sr;
    p.x = xr.ptr; p.x_stride = xr.stride;
    if (shortcut) { sr = Rows(*shortcut); p.shortcut = sr.ptr; p.shortcut_stride = sr.stride; }
    p.y = ptr(o.y); p.h = ptr(o.h); p.y8 = ptr(o.y8); p.y8_scale = (float*)ptr(o.scale); p.stats = (float*)ptr(o.stats);
    p.stream = stream_of(x);
    check(fwa2_norm_forward(&p), "fwa2_norm_forward");
    return o;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Optional& shortcut, const Optional& bias,
                                 const Optional& gate, const NormHow& how) {
        const NormOut o = norm_forward(x, shortcut, weight, bias, gate, how, true, false);
        // kept for the backward pass: x (post), the h returned (pre over an fp32 stream) or x and shortcut (pre over a 16-bit
        // one, whose h was rounded), and two numbers per row
        ctx->save_for_backward({how.exact_h() ? o.h : x, weight, value(bias), value(gate), o.stats, how.two() ? value(shortcut) : Tensor()});
        ctx->saved_data["eps"] = how.eps;
        ctx->saved_data["how"] = (int64_t)(how.kind + 2 * how.place + 4 * (shortcut ? 1 : 0) + 8 * (bias ? 1 : 0) + 16 * (int)how.x + 4096 * (int)how.stream);
        ctx->set_materialize_grads(false);
        if (how.pre()) return {o.h, o.y};
        return {o.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &v = saved[0], &weight = saved[1], &bias = saved[2], &gate = saved[3], &stats = saved[4], &shortcut = saved[5];
        const int64_t code = ctx->saved_data["how"].toInt();
        const NormHow how = {ctx->saved_data["eps"].toDouble(), (int)(code & 1), (int)(code >> 1 & 1), (at::ScalarType)(code / 16 % 256),
                             (at::ScalarType)(code / 4096)};
        const bool has_s = code & 4, has_b = code & 8;
        const Tensor dy = how.pre() ? grads[1] : grads[0], dh = how.pre() ? grads[0] : Tensor();
        if (!dy.defined() && !dh.defined()) return variable_list(6);
        refuse_unseen(dy, dh);
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1) && dy.defined(), need_s = has_s && ctx->needs_input_grad(2),
                   need_b = has_b && ctx->needs_input_grad(2 + has_s) && dy.defined();
        Tensor dx, ds, dw, db;
        // without a gate and with one type, the two gradients of the pre-norm form are the same numbers
        const bool shared = how.pre() && !gate.defined() && how.x == how.stream;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const c10::DeviceGuard guard(v.device());
            if (how.pre() && (need_s || (shared && need_x))) ds = make(v.sizes(), v, how.stream);
            if (need_x && !shared) dx = make(v.sizes(), v, how.x);
            if (need_w) dw = make(weight.sizes(), v, weight.scalar_type());
            if (need_b) db = make(bias.sizes(), v, bias.scalar_type());
            if (row_count(v) == 0) {
                if (dw.defined()) dw.zero_();
                if (db.defined()) db.zero_();
            } else if (dx.defined() || ds.defined() || dw.defined() || db.defined()) {
                NormParams keep;
                fwa2_norm p = norm_description(v, how, weight, bias, gate, keep);
                Rows vr, sr, dyr, dhr;
                if (how.exact_h()) {
                    p.h = ptr(v);       // an output of the forward call: contiguous
                } else {
                    vr = Rows(v);
                    p.x = vr.ptr; p.x_stride = vr.stride;
                }
                if (how.two()) { sr = Rows(shortcut); p.shortcut = sr.ptr; p.shortcut_stride = sr.stride; }
                if (dh.defined()) { dhr = Rows(dh); p.dh = dhr.ptr; p.dh_stride = dhr.stride; }
                if (dy.defined()) { dyr = Rows(dy); p.dy = dyr.ptr; p.dy_stride = dyr.stride; }
                p.stats = (float*)ptr(stats);
                p.dx = ptr(dx); p.dshortcut = ptr(ds); p.dweight = ptr(dw); p.dbias = ptr(db);
                Tensor ws;
                if (const size_t need = fwa2_norm_workspace_bytes(&p)) {
                    ws = make({(int64_t)need}, v, at::kByte);
                    p.workspace = ws.data_ptr();
                    p.workspace_bytes = need;
                }
                p.stream = stream_of(v);
                check(fwa2_norm_backward(&p), "fwa2_norm_backward");
            }
        }
        if (shared && need_x) dx = ds;
        if (!how.pre()) ds = dy;
        return once({dx, dw, need_s ? ds : Tensor(), db, Tensor(), Tensor()});
    }
};

NormHow norm_how(const Tensor& x, const Optional& shortcut, double eps, int64_t kind, int64_t place) {
    return {eps, (int)kind, (int)place, x.scalar_type(), shortcut ? shortcut->scalar_type() : x.scalar_type()};
}

// [y] (post) or [h, y] (pre)
variable_list norm(const Tensor& x, const Optional& shortcut, const Tensor& weight, const Optional& bias, double eps, int64_t kind, int64_t place,
                   const Optional& gate) {
    refuse_unseen(x, shortcut, weight, bias, gate);
    const NormHow how = norm_how(x, shortcut, eps, kind, place);
    const Optional xo(x), wo(weight);
    if (wants_grad({&xo, &wo, &shortcut, &bias})) return NormNode::apply(x, weight, shortcut, bias, gate, how);
    const NormOut o = norm_forward(x, shortcut, weight, bias, gate, how, false, false);
    if (how.pre()) return {o.h, o.y};
    return {o.y};
}

// [stream, y8, scale]
variable_list norm_fp8(const Tensor& x, const Optional& shortcut, const Tensor& weight, const Optional& bias, double eps, int64_t kind, int64_t place,
                       const Optional& gate) {
    refuse_unseen(x, shortcut, weight, bias, gate);
    const NormHow how = norm_how(x, shortcut, eps, kind, place);
    const NormOut o = norm_forward(x, shortcut, weight, bias, gate, how, false, true);
    return {how.pre() ? o.h : o.y, o.y8, o.scale};
}

std::pair<Tensor, Tensor> quantize_rows(const Tensor& x) {
    refuse_unseen(x);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    Tensor x8 = make(x.sizes(), x, at::kFloat8_e4m3fn), scale = make(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
    const int64_t rows = row_count(x);
    if (rows == 0) return {x8, scale};
    const Rows xr(x);
    check(fwa2_quantize_rows(xr.ptr, dtype_code(x.scalar_type()), rows, (int)x.size(-1), xr.stride, x8.data_ptr(), scale.data_ptr<float>(),
                             stream_of(x)),
          "fwa2_quantize_rows");
    return {x8, scale};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr e) {
        try {
            if (e) std::rethrow_exception(e);
        } catch (const StatusError& s) {
            PyObject* type = s.code == FWA2_ERR_INVALID_ARGUMENT ? PyExc_AssertionError
                             : s.code == FWA2_ERR_UNSUPPORTED    ? PyExc_NotImplementedError
                                                                 : PyExc_RuntimeError;
            PyErr_SetString(type, s.what());
        }
    });
    m.def("abi_version", [] { return FWA2_ABI_VERSION; });
    m.def("linear", &linear);
    m.def("linear_fp8", &linear_fp8);
    m.def("norm", &norm);
    m.def("norm_fp8", &norm_fp8);
    m.def("quantize_rows", &quantize_rows);
    m.def("rows", [](const Tensor& t) { const Rows r(t); return std::make_pair(r.t.reshape({-1, t.size(-1)}), r.stride); });
}
