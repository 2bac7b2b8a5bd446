// torch_ops.cpp — the operators of include/sdengine.h on torch tensors, with autograd (diffusers_amd/_torch_ops.so).
//
// In C++ because a backward pass runs on autograd's own thread: written in Python it cost 100 us a call there (measured on a 2 x 1280 layer norm, forward and
// gradients: 140 us), several times what the kernels take.  The library's entry points come from Python as addresses (bind), so that
// both sides use one copy of it.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/sdengine.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Entries {
    decltype(&sde_last_error) last_error;
    decltype(&sde_layer_norm_forward) ln_forward;
    decltype(&sde_layer_norm_backward) ln_backward;
    decltype(&sde_layer_norm_workspace) ln_workspace;
    decltype(&sde_gated_ff_forward) ff_forward;
    decltype(&sde_gated_ff_backward) ff_backward;
    decltype(&sde_gated_ff_workspace) ff_workspace;
    decltype(&sde_cross_attention_forward) xa_forward;
    decltype(&sde_cross_attention_backward) xa_backward;
    decltype(&sde_cross_attention_workspace) xa_workspace;
} entry;

struct StatusError : std::runtime_error {          // becomes _lib.SdeError
    int status;
    StatusError(int s, const char* m) : std::runtime_error(m), status(s) {}
};
void done(sde_status s)
{
    if (s != SDE_OK) throw StatusError(s, entry.last_error());
}
[[noreturn]] void bad_value(const std::string& m) { throw py::value_error(m); }
[[noreturn]] void bad_type(const std::string& m) { throw py::type_error(m); }
template <typename... A> std::string text(const A&... a) { return c10::str(a...); }

int dtype_of(const Tensor& t)
{
    switch (t.scalar_type()) {
    case at::kHalf: return SDE_F16;
    case at::kBFloat16: return SDE_BF16;
    case at::kFloat: return SDE_F32;
    default: return -1;
    }
}
void first_tensor(const Tensor& x)
{
    if (!x.defined() || !x.is_cuda()) bad_value("the operators take tensors on a GPU");
    if (dtype_of(x) < 0) bad_type(text("fp16, bf16 or fp32 tensors, not ", x.scalar_type()));
}
void beside(const Tensor& t, const Tensor& x, const char* name)
{
    if (t.defined() && t.device() != x.device()) bad_value(text(name, " is on ", t.device(), ", the first tensor on ", x.device()));
}
Tensor or_none(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// x as rows of `cols` contiguous values, every row on `align` bytes and apart from the others; copied where it has to be
Tensor as_rows(Tensor x, int64_t cols, int64_t align)
{
    if (x.dim() != 2) x = x.reshape({x.numel() / cols, cols});
    const int64_t e = x.element_size(), n = x.size(0);
    if ((cols > 1 && x.stride(1) != 1) || (n > 1 && x.stride(0) < cols)) x = x.contiguous();
    if (align > 1 && ((uintptr_t)x.data_ptr() % align || (n > 1 && (x.stride(0) * e % align || x.stride(0) * e >= (1 << 23))))) x = x.clone(at::MemoryFormat::Contiguous);
    return x;
}
int64_t ld(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

struct Exec {                                       // the current stream of the tensors' device, and scratch on it
    Tensor scratch;
    sde_op_exec e{};
    explicit Exec(const Tensor& like, size_t bytes = 0)
    {
        e.device_id = like.device().index();
        e.hip_stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.device().index()).stream();
        if (bytes) {
            scratch = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
            e.workspace = scratch.data_ptr();
            e.workspace_bytes = bytes;
        }
    }
};
// autograd takes no tensor that is not there: one that was left out goes in as x (and gets no gradient), with a mark
const Tensor& or_x(const Tensor& t, const Tensor& x) { return t.defined() ? t : x; }
struct Given { bool weight, bias; };
// A backward pass captured into a graph ends the process if the node that gathers a leaf's gradient still belongs to another stream, as it does while a graph built
// outside of the capture lives: refused here, where the capture can still be given up in order.
void leaves_of_this_capture(const Tensor& like, std::initializer_list<const Tensor*> inputs)
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const c10::Stream here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.device().index()).unwrap();
    for (const Tensor* t : inputs) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (node && node->stream() && *node->stream() != here)
            throw std::runtime_error("this call is being captured, and a graph of the same leaves that was built on another stream is alive: let go of it first");
    }
}
// forward-mode differentiation: a tangent would be left behind without a word
void no_tangent(std::initializer_list<const Tensor*> inputs)
{
    for (const Tensor* t : inputs)
        if (t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error("the operators have no forward-mode derivatives: an argument carries a tangent");
}
// gradients come from kernels autograd does not see: a graph through them would be wrong
void first_derivative_only(const Tensor& upstream)
{
    no_tangent({&upstream});
    if (at::GradMode::is_enabled()) throw std::runtime_error("the operators have first derivatives only (create_graph is set)");
}

// ------------------------------------------------------------------------------------------ layer norm
sde_layer_norm_args ln_args(const Tensor& x2, const Tensor& weight, const Tensor& bias, double eps)
{
    sde_layer_norm_args a{};
    a.dtype = dtype_of(x2);
    a.param_dtype = weight.defined() ? dtype_of(weight) : bias.defined() ? dtype_of(bias) : a.dtype;
    a.rows = x2.size(0);
    a.C = x2.size(1);
    a.ld_x = ld(x2);
    a.ld_y = a.ld_dx = a.C;
    a.eps = (float)eps;
    a.x = ptr(x2);
    a.gamma = ptr(weight);
    a.beta = ptr(bias);
    return a;
}
Tensor ln_forward(const Tensor& x, const Tensor& x2, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats)
{
    Tensor y = at::empty(x.sizes(), x.options());
    sde_layer_norm_args a = ln_args(x2, weight, bias, eps);
    a.y = ptr(y);
    if (stats) {
        *stats = at::empty({2, a.rows}, x.options().dtype(at::kFloat));
        a.mean = (float*)stats->data_ptr();
        a.rstd = a.mean + a.rows;
        if (!a.rows) a.mean = a.rstd = nullptr;
    }
    Exec ex(x);
    done(entry.ln_forward(&a, &ex.e));
    return y;
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& b, Given given, double eps)
    {
        const Tensor weight = given.weight ? w : Tensor(), bias = given.bias ? b : Tensor();
        Tensor stats, x2 = as_rows(x, x.size(-1), 1);
        Tensor y = ln_forward(x, x2, weight, bias, eps, &stats);
        ctx->save_for_backward({x2, weight, bias, stats});
        ctx->saved_data["eps"] = eps;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        first_derivative_only(grads[0]);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x2 = s[0], &weight = s[1], &bias = s[2], &stats = s[3], &dy = grads[0];
        const Tensor d2 = as_rows(dy, x2.size(1), 1);
        Tensor dx, dw, db;
        if (ctx->needs_input_grad(0)) dx = at::empty(dy.sizes(), x2.options());
        if (weight.defined() && ctx->needs_input_grad(1)) dw = at::empty(weight.sizes(), weight.options());
        if (bias.defined() && ctx->needs_input_grad(2)) db = at::empty(bias.sizes(), bias.options());
        sde_layer_norm_args a = ln_args(x2, weight, bias, ctx->saved_data["eps"].toDouble());
        a.mean = (float*)ptr(stats);
        a.rstd = a.rows ? a.mean + a.rows : nullptr;
        a.ld_dy = ld(d2);
        a.dy = ptr(d2);
        a.dx = ptr(dx);
        a.dgamma = ptr(dw);
        a.dbeta = ptr(db);
        size_t n = 0;
        done(entry.ln_workspace(&a, &n));
        Exec ex(x2, n);
        done(entry.ln_backward(&a, &ex.e));
        return {dx, dw, db, Tensor(), Tensor()};
    }
};
Tensor param(const Tensor& p, const Tensor& x, int64_t n, const char* name)
{
    if (!p.defined()) return p;
    if (p.dim() != 1 || p.size(0) != n) bad_value(text(name, " has shape ", p.sizes(), ", not [", n, "]"));
    if (p.scalar_type() != x.scalar_type() && p.scalar_type() != at::kFloat) bad_type(text(name, " is ", p.scalar_type(), ": ", x.scalar_type(), " or Float"));
    return p.contiguous();
}
Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, double eps)
{
    first_tensor(x);
    Tensor weight = or_none(weight_), bias = or_none(bias_);
    beside(weight, x, "weight");
    beside(bias, x, "bias");
    if (x.dim() == 0 || x.size(-1) == 0) bad_value("layer_norm needs a last axis that is not empty");
    no_tangent({&x, &weight, &bias});
    const int64_t c = x.size(-1);
    weight = param(weight, x, c, "weight");
    bias = param(bias, x, c, "bias");
    if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type()) bad_type("weight and bias have one type");
    if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias))) {
        leaves_of_this_capture(x, {&x, &weight, &bias});
        return LayerNorm::apply(x, or_x(weight, x), or_x(bias, x), Given{weight.defined(), bias.defined()}, eps);
    }
    return ln_forward(x, as_rows(x, c, 1), weight, bias, eps, nullptr);
}

// ------------------------------------------------------------------------------------------ gated feed-forward
sde_gated_ff_args ff_args(const Tensor& x2, const Tensor& w2, const Tensor& bias, int64_t act)
{
    sde_gated_ff_args a{};
    a.dtype = dtype_of(x2);
    a.bias_dtype = bias.defined() ? dtype_of(bias) : a.dtype;
    a.activation = (int)act;
    a.M = x2.size(0);
    a.K = x2.size(1);
    a.F = w2.size(0) / 2;
    a.ld_x = ld(x2);
    a.ld_w = ld(w2);
    a.ld_h = a.F;
    a.ld_dx = a.ld_dw = a.K;
    a.x = ptr(x2);
    a.weight = ptr(w2);
    a.bias = ptr(bias);
    return a;
}
Tensor ff_forward(const Tensor& x, const Tensor& x2, const Tensor& w2, const Tensor& bias, int64_t act)
{
    sde_gated_ff_args a = ff_args(x2, w2, bias, act);
    c10::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = a.F;
    Tensor h = at::empty(shape, x.options());
    a.h = ptr(h);
    size_t n = 0;
    done(entry.ff_workspace(&a, 0, &n));
    Exec ex(x, n);
    done(entry.ff_forward(&a, &ex.e));
    return h;
}
struct GatedFf : torch::autograd::Function<GatedFf> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& b, Given given, int64_t act)
    {
        const Tensor bias = given.bias ? b : Tensor();
        const Tensor x2 = as_rows(x, x.size(-1), 16), w2 = as_rows(weight, weight.size(1), 16);
        ctx->save_for_backward({x2, w2, bias});
        ctx->saved_data["act"] = act;
        return ff_forward(x, x2, w2, bias, act);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        first_derivative_only(grads[0]);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x2 = s[0], &w2 = s[1], &bias = s[2], &dh = grads[0];
        sde_gated_ff_args a = ff_args(x2, w2, bias, ctx->saved_data["act"].toInt());
        const Tensor d2 = as_rows(dh, a.F, 16);
        Tensor dx, dw, db;
        if (ctx->needs_input_grad(0)) {
            c10::DimVector shape(dh.sizes().begin(), dh.sizes().end());
            shape.back() = a.K;
            dx = at::empty(shape, x2.options());
        }
        if (ctx->needs_input_grad(1)) dw = at::empty({2 * a.F, a.K}, w2.options());
        if (bias.defined() && ctx->needs_input_grad(2)) db = at::empty(bias.sizes(), bias.options());
        a.ld_dh = ld(d2);
        a.dh = ptr(d2);
        a.dx = ptr(dx);
        a.dweight = ptr(dw);
        a.dbias = ptr(db);
        size_t n = 0;
        done(entry.ff_workspace(&a, 1, &n));
        Exec ex(x2, n);
        done(entry.ff_backward(&a, &ex.e));
        return {dx, dw, db, Tensor(), Tensor()};
    }
};
Tensor gated_ff(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_, int64_t act)
{
    first_tensor(x);
    beside(weight, x, "weight");
    Tensor bias = or_none(bias_);
    beside(bias, x, "bias");
    const int64_t step = 16 / x.element_size();
    if (x.dim() == 0 || weight.dim() != 2 || weight.size(1) != x.size(-1) || weight.size(0) % 2)
        bad_value(text("x [..., K] and weight [2F, K], not ", x.sizes(), " and ", weight.sizes()));
    if (weight.scalar_type() != x.scalar_type()) bad_type(text("weight is ", weight.scalar_type(), ", x is ", x.scalar_type()));
    const int64_t k = x.size(-1), f = weight.size(0) / 2;
    if (!k || !f || k % step || f % step) bad_value(text("K and F are positive multiples of ", step, " for ", x.scalar_type()));
    no_tangent({&x, &weight, &bias});
    bias = param(bias, x, 2 * f, "bias");
    if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias))) {
        leaves_of_this_capture(x, {&x, &weight, &bias});
        return GatedFf::apply(x, weight, or_x(bias, x), Given{true, bias.defined()}, act);
    }
    return ff_forward(x, as_rows(x, k, 16), as_rows(weight, k, 16), bias, act);
}

// ------------------------------------------------------------------------------------------ cross attention
// x [B, S, H, D] as the kernels take it: last axis contiguous, every (b, s, h) on 16 bytes, offsets inside a tile within 2 GB
Tensor as_heads(const Tensor& x)
{
    const int64_t e = x.element_size(), step = 16 / e;
    if (x.stride(3) != 1 || x.stride(0) % step || x.stride(1) % step || x.stride(2) % step || (uintptr_t)x.data_ptr() % 16 ||
        (65 * x.stride(1) + x.size(2) * x.stride(2) + x.size(3)) * e >= (int64_t(1) << 31))
        return x.clone(at::MemoryFormat::Contiguous);
    return x;
}
void strides(int64_t (&s)[3], const Tensor& t)
{
    if (t.defined())
        for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}
sde_cross_attention_args xa_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& q_lens,
                                 const Tensor& kv_lens, const Tensor& mask, double scale)
{
    sde_cross_attention_args a{};
    a.dtype = dtype_of(q);
    a.B = q.size(0);
    a.Sq = q.size(1);
    a.H = q.size(2);
    a.D = q.size(3);
    a.Skv = k.size(1);
    a.Hkv = k.size(2);
    a.scale = (float)scale;
    a.q = ptr(q);
    a.k = ptr(k);
    a.v = ptr(v);
    a.o = ptr(o);
    a.lse = (float*)ptr(lse);
    a.q_lens = (const int32_t*)ptr(q_lens);
    a.kv_lens = (const int32_t*)ptr(kv_lens);
    a.key_mask = (const uint8_t*)ptr(mask);
    a.key_mask_stride = mask.defined() ? mask.stride(0) : 0;
    strides(a.q_stride, q);
    strides(a.k_stride, k);
    strides(a.v_stride, v);
    strides(a.o_stride, o);
    return a;
}
Tensor xa_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_lens, const Tensor& kv_lens, const Tensor& mask, double scale, Tensor* lse)
{
    Tensor o = at::empty(q.sizes(), q.options());
    if (lse) *lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    sde_cross_attention_args a = xa_args(q, k, v, o, lse ? *lse : Tensor(), q_lens, kv_lens, mask, scale);
    size_t n = 0;
    done(entry.xa_workspace(&a, 0, &n));
    Exec ex(q, n);
    done(entry.xa_forward(&a, &ex.e));
    return o;
}
struct Counts { Tensor q_lens, kv_lens, mask; };      // each may be undefined; no gradients
struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Counts& n, double scale)
    {
        const Tensor q = as_heads(q_), k = as_heads(k_), v = as_heads(v_);
        Tensor lse, o = xa_forward(q, k, v, n.q_lens, n.kv_lens, n.mask, scale, &lse);
        ctx->save_for_backward({q, k, v, o, lse, n.q_lens, n.kv_lens, n.mask});
        ctx->saved_data["scale"] = scale;
        return o;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        first_derivative_only(grads[0]);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2];
        const Tensor d_o = as_heads(grads[0]);
        sde_cross_attention_args a = xa_args(q, k, v, s[3], s[4], s[5], s[6], s[7], ctx->saved_data["scale"].toDouble());
        Tensor dq, dk, dv;
        if (ctx->needs_input_grad(0)) dq = at::empty(q.sizes(), q.options());
        if (ctx->needs_input_grad(1)) dk = at::empty(k.sizes(), k.options());
        if (ctx->needs_input_grad(2)) dv = at::empty(v.sizes(), v.options());
        a.d_o = ptr(d_o);
        a.dq = ptr(dq);
        a.dk = ptr(dk);
        a.dv = ptr(dv);
        strides(a.do_stride, d_o);
        strides(a.dq_stride, dq);
        strides(a.dk_stride, dk);
        strides(a.dv_stride, dv);
        size_t n = 0;
        done(entry.xa_workspace(&a, 1, &n));
        Exec ex(q, n);
        done(entry.xa_backward(&a, &ex.e));
        return {dq, dk, dv, Tensor(), Tensor()};
    }
};
Tensor lengths(const Tensor& t, int64_t b, const char* name)
{
    if (!t.defined()) return t;
    if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.dim() != 1 || t.size(0) != b)
        bad_value(text(name, " is an int32 (or int64) tensor of shape [", b, "]"));
    return (t.scalar_type() == at::kLong ? t.clamp(0, INT32_MAX).to(at::kInt) : t).contiguous();
}
Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& q_lens_, const std::optional<Tensor>& kv_lens_,
                       const std::optional<Tensor>& mask_, std::optional<double> scale_)
{
    first_tensor(q);
    Tensor q_lens = or_none(q_lens_), kv_lens = or_none(kv_lens_), mask = or_none(mask_);
    beside(k, q, "k");
    beside(v, q, "v");
    beside(q_lens, q, "q_lens");
    beside(kv_lens, q, "kv_lens");
    beside(mask, q, "key_mask");
    if (q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
        bad_value(text("q [B, Sq, H, D] and k, v [B, Skv, Hkv, D], not ", q.sizes(), ", ", k.sizes(), ", ", v.sizes()));
    if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) bad_type("q, k and v have one type");
    const int64_t b = q.size(0), h = q.size(2), d = q.size(3), hk = k.size(2), skv = k.size(1), step = 16 / q.element_size();
    if (!h || !hk || h % hk || d <= 0 || d > 256 || d % step)
        bad_value(text("H is a multiple of Hkv, and D at most 256 and a multiple of ", step, " for ", q.scalar_type()));
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)d);
    if (!(scale > 0.0) || !std::isfinite((float)scale * 1.5f)) bad_value("scale is positive and finite");
    no_tangent({&q, &k, &v});
    q_lens = lengths(q_lens, b, "q_lens");
    kv_lens = lengths(kv_lens, b, "kv_lens");
    if (mask.defined()) {
        if ((mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte) || mask.dim() != 2 || mask.size(0) != b || mask.size(1) != skv)
            bad_value(text("key_mask is a bool tensor of shape [", b, ", ", skv, "]"));
        if ((skv > 1 && mask.stride(1) != 1) || (b > 1 && mask.stride(0) < skv)) mask = mask.contiguous();
    }
    if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v))) {
        leaves_of_this_capture(q, {&q, &k, &v});
        return CrossAttention::apply(q, k, v, Counts{q_lens, kv_lens, mask}, scale);
    }
    return xa_forward(as_heads(q), as_heads(k), as_heads(v), q_lens, kv_lens, mask, scale, nullptr);
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m)
{
    m.def("bind", [](const py::dict& at, py::object error) {
        auto take = [&](auto& f, const char* name) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at[name].cast<uintptr_t>()); };
        take(entry.last_error, "sde_last_error");
        take(entry.ln_forward, "sde_layer_norm_forward");
        take(entry.ln_backward, "sde_layer_norm_backward");
        take(entry.ln_workspace, "sde_layer_norm_workspace");
        take(entry.ff_forward, "sde_gated_ff_forward");
        take(entry.ff_backward, "sde_gated_ff_backward");
        take(entry.ff_workspace, "sde_gated_ff_workspace");
        take(entry.xa_forward, "sde_cross_attention_forward");
        take(entry.xa_backward, "sde_cross_attention_backward");
        take(entry.xa_workspace, "sde_cross_attention_workspace");
        static PyObject* type = error.release().ptr();           // _lib.SdeError, kept for the process
        py::register_local_exception_translator([](std::exception_ptr p) {
            try {
                if (p) std::rethrow_exception(p);
            } catch (const StatusError& e) {
                const py::object err = py::reinterpret_borrow<py::object>(type)(e.status, e.what());
                PyErr_SetObject(type, err.ptr());
            }
        });
    });
    m.def("layer_norm", &layer_norm);
    m.def("gated_ff", &gated_ff);
    m.def("cross_attention", &cross_attention);
}
