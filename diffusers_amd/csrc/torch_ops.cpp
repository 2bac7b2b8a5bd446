// torch_ops.cpp — the operators of include/sdengine.h on torch tensors, with autograd (diffusers_amd/_torch_ops.so).
//
// In C++ because a backward pass runs on autograd's own thread: written in Python it cost 100 us a call there (measured on a 2 x 1280 layer norm, forward and
// gradients: 140 us), several times what the kernels take.  The library's entry points come from Python as addresses (bind), so that
// both sides use one copy of it.
//
// Every launch stands inside an operator registered with torch's dispatcher (torch.ops.diffusers_amd): tracers record it as one node, where a plain function that fills
// the memory of a fresh tensor would leave them a graph that returns that tensor unfilled.  The Autograd entries hold the gradients, the CUDA entries launch, and the Meta entries,
// which are the same functions, give shapes alone.
#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <unordered_set>

#include "../../include/sdengine.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;
typedef std::array<bool, 3> Wanted;                // which gradients a backward pass forms; the others come back undefined

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
PyObject* sde_error = nullptr;                     // _lib.SdeError, kept for the process

// A refusal of the library becomes _lib.SdeError, on whichever thread it happens (autograd hands it on).
void done(sde_status s)
{
    if (s == SDE_OK) return;
    const std::string message = entry.last_error();
    py::gil_scoped_acquire gil;
    const py::object type = py::reinterpret_borrow<py::object>(sde_error);
    PyErr_SetObject(sde_error, type((int)s, message).ptr());
    python_error e;
    e.persist();
    throw e;
}
[[noreturn]] void bad_value(const std::string& m) { TORCH_CHECK_VALUE(false, m); }
[[noreturn]] void bad_type(const std::string& m) { TORCH_CHECK_TYPE(false, m); }
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
void on_a_gpu(const Tensor& x)
{
    if (!x.defined() || !x.is_cuda()) bad_value("the operators take tensors on a GPU");
}
void first_tensor(const Tensor& x)
{
    TORCH_CHECK(entry.last_error, "the operators are reached through diffusers_amd.ops");
    if (dtype_of(x) < 0) bad_type(text("fp16, bf16 or fp32 tensors, not ", x.scalar_type()));
}
void beside(const Tensor& t, const Tensor& x, const char* name)
{
    if (t.defined() && t.device() != x.device()) bad_value(text(name, " is on ", t.device(), ", the first tensor on ", x.device()));
}
Tensor or_none(const MaybeTensor& t) { return t ? *t : Tensor(); }
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }
void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const MaybeTensor& t) { return t && wants(*t); }

// Tensors without memory (shapes alone, a tracer's) count as aligned: the launch looks again.
bool has_memory(const Tensor& x) { return !x.is_meta() && (x.key_set() & at::kTensorSubclassLike).empty(); }
bool aligned(const Tensor& x, int64_t align) { return align == 1 || !has_memory(x) || (uintptr_t)x.data_ptr() % align == 0; }

// x [..., cols] as rows: elements from row to row, -1 where the leading axes have no one step
int64_t row_step(const Tensor& x)
{
    int64_t n = 1, step = x.size(-1);
    for (int64_t d = x.dim() - 2; d >= 0; --d) {
        if (x.size(d) == 1) continue;
        if (n == 1) step = x.stride(d);
        else if (x.stride(d) != step * n) return -1;
        n *= x.size(d);
    }
    return step;
}
// x as rows of contiguous values, every row on `align` bytes and apart from the others; copied where it has to be
Tensor as_rows(const Tensor& x, int64_t align)
{
    const int64_t cols = x.size(-1), e = x.element_size(), step = row_step(x);
    if (x.numel() == 0) return x;
    if ((cols > 1 && x.stride(-1) != 1) || step < cols) return x.clone(at::MemoryFormat::Contiguous);
    if (align > 1 && (!aligned(x, align) || step * e % align || step * e >= (1 << 23))) return x.clone(at::MemoryFormat::Contiguous);
    return x;
}
int64_t rows_of(const Tensor& x) { return x.numel() / x.size(-1); }
int64_t ld(const Tensor& x) { return x.numel() ? row_step(x) : x.size(-1); }

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
const Tensor& or_x(const MaybeTensor& t, const Tensor& x) { return t ? *t : x; }
struct Given { bool weight, bias; };
// A backward pass captured into a graph ends the process if a gradient goes to a node that belongs to another stream, as the node that gathers a leaf's gradient does while a graph
// built outside of the capture lives: refused, where the capture can still be given up in order.
bool capturing(const Tensor& like)
{
    if (!has_memory(like)) return false;
    const c10::OptionalDeviceGuard on(like.device());          // the status is that of the current device's current stream
    return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}
c10::Stream stream_of(const Tensor& like) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.device().index()).unwrap(); }
bool elsewhere(torch::autograd::Node* node, c10::Stream here) { return node->stream() && *node->stream() != here; }
// In the forward pass: the leaves of `inputs`, also those behind views and other steps of this capture.  Steps from outside of it are not looked through: whether
// their gradients will be asked for is known in the backward pass (below).
void leaves_of_this_capture(const Tensor& like, std::initializer_list<Tensor> inputs)
{
    if (!capturing(like)) return;
    const c10::Stream here = stream_of(like);
    std::vector<std::shared_ptr<torch::autograd::Node>> nodes;
    std::unordered_set<const torch::autograd::Node*> seen;
    for (const Tensor& t : inputs)
        if (t.defined() && t.requires_grad()) nodes.push_back(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
    while (!nodes.empty()) {
        const auto node = nodes.back();
        nodes.pop_back();
        if (!node || !seen.insert(node.get()).second) continue;
        const bool other = elsewhere(node.get(), here);
        if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) {
            if (other) throw std::runtime_error("this call is being captured, and a graph of the same leaves that was built on another stream is alive: let go of it first");
        } else if (!other) {
            for (const auto& edge : node->next_edges()) nodes.push_back(edge.function);
        }
    }
}
// In the backward pass: a gradient for a step that was taken outside of the capture.
void steps_of_this_capture(const Tensor& upstream)
{
    if (!capturing(upstream)) return;
    const c10::Stream here = stream_of(upstream);
    const auto node = torch::autograd::get_current_node();
    for (size_t i = 0; node && i < node->num_outputs(); ++i) {
        const auto& edge = node->next_edge(i);
        if (edge.is_valid() && node->task_should_compute_output(i) && elsewhere(edge.function.get(), here))
            throw std::runtime_error("this backward pass is being captured, and it reaches a step that was taken on another stream: take the whole forward pass inside the capture, or detach()");
    }
}
// forward-mode differentiation: a tangent would be left behind without a word
void no_tangent(std::initializer_list<Tensor> inputs)
{
    for (const Tensor& t : inputs)
        if (t.defined() && t._fw_grad(0).defined()) throw std::runtime_error("the operators have no forward-mode derivatives: an argument carries a tangent");
}
// In front of every backward pass.  Gradients come from kernels autograd does not see: a graph through them would be wrong
void check_backward(const Tensor& upstream)
{
    no_tangent({upstream});
    steps_of_this_capture(upstream);
    if (at::GradMode::is_enabled()) throw std::runtime_error("the operators have first derivatives only (create_graph is set)");
}
// Calls an operator through the dispatcher; `Below`: its CUDA or Meta entry (or a tracer in front of it), not its Autograd entry.
template <typename F> c10::TypedOperatorHandle<F> op(const char* name) { return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>(); }
typedef at::AutoDispatchBelowADInplaceOrView Below;

// ------------------------------------------------------------------------------------------ layer norm
Tensor param(const Tensor& p, const Tensor& x, int64_t n, const char* name)
{
    if (!p.defined()) return p;
    if (p.dim() != 1 || p.size(0) != n) bad_value(text(name, " has shape ", p.sizes(), ", not [", n, "]"));
    if (p.scalar_type() != x.scalar_type() && p.scalar_type() != at::kFloat) bad_type(text(name, " is ", p.scalar_type(), ": ", x.scalar_type(), " or Float"));
    return p.contiguous();
}
struct LnInputs { Tensor x, weight, bias; sde_layer_norm_args a{}; };
LnInputs ln_inputs(const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, double eps)
{
    first_tensor(x);
    LnInputs in;
    beside(in.weight = or_none(weight_), x, "weight");
    beside(in.bias = or_none(bias_), x, "bias");
    if (x.dim() == 0 || x.size(-1) == 0) bad_value("layer_norm needs a last axis that is not empty");
    in.weight = param(in.weight, x, x.size(-1), "weight");
    in.bias = param(in.bias, x, x.size(-1), "bias");
    if (in.weight.defined() && in.bias.defined() && in.weight.scalar_type() != in.bias.scalar_type()) bad_type("weight and bias have one type");
    in.x = as_rows(x, 1);
    sde_layer_norm_args& a = in.a;
    a.dtype = dtype_of(x);
    a.param_dtype = in.weight.defined() ? dtype_of(in.weight) : in.bias.defined() ? dtype_of(in.bias) : a.dtype;
    a.rows = rows_of(x);
    a.C = x.size(-1);
    a.ld_x = ld(in.x);
    a.ld_y = a.ld_dx = a.C;
    a.eps = (float)eps;
    if (x.is_meta()) return in;
    a.x = ptr(in.x);
    a.gamma = ptr(in.weight);
    a.beta = ptr(in.bias);
    return in;
}
Tensor ln_forward(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, Tensor* stats)
{
    LnInputs in = ln_inputs(x, weight, bias, eps);
    Tensor y = at::empty(x.sizes(), x.options());
    if (stats) *stats = at::empty({2, in.a.rows}, x.options().dtype(at::kFloat));
    if (x.is_meta()) return y;
    in.a.y = ptr(y);
    if (stats && in.a.rows) {
        in.a.mean = (float*)stats->data_ptr();
        in.a.rstd = in.a.mean + in.a.rows;
    }
    Exec ex(x);
    done(entry.ln_forward(&in.a, &ex.e));
    return y;
}
Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) { return ln_forward(x, weight, bias, eps, nullptr); }
std::tuple<Tensor, Tensor> layer_norm_kept(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps)
{
    Tensor stats, y = ln_forward(x, weight, bias, eps, &stats);
    return {y, stats};
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& dy, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, const Tensor& stats,
                                                       double eps, Wanted wanted)
{
    LnInputs in = ln_inputs(x, weight, bias, eps);
    sde_layer_norm_args& a = in.a;
    Tensor dx, dw, db;
    if (wanted[0]) dx = at::empty(x.sizes(), x.options());
    if (wanted[1]) dw = at::empty(in.weight.sizes(), in.weight.options());
    if (wanted[2]) db = at::empty(in.bias.sizes(), in.bias.options());
    if (x.is_meta()) return {dx, dw, db};
    const Tensor d2 = as_rows(dy, 1);
    a.mean = (float*)ptr(stats);
    a.rstd = a.rows ? a.mean + a.rows : nullptr;
    a.ld_dy = ld(d2);
    a.dy = ptr(d2);
    a.dx = ptr(dx);
    a.dgamma = ptr(dw);
    a.dbeta = ptr(db);
    size_t n = 0;
    done(entry.ln_workspace(&a, &n));
    Exec ex(x, n);
    done(entry.ln_backward(&a, &ex.e));
    return {dx, dw, db};
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w, const Tensor& b, Given given, double eps)
    {
        static const auto kept = op<std::tuple<Tensor, Tensor>(const Tensor&, const MaybeTensor&, const MaybeTensor&, double)>("diffusers_amd::_layer_norm_kept");
        Below below;
        const Tensor x = x_.dim() && x_.size(-1) ? as_rows(x_, 1) : x_, weight = given.weight ? w : Tensor(), bias = given.bias ? b : Tensor();
        auto [y, stats] = kept.call(x, maybe(weight), maybe(bias), eps);
        ctx->save_for_backward({x, weight, bias, stats});
        ctx->saved_data["eps"] = eps;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        static const auto back = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&, const Tensor&, double, Wanted)>(
            "diffusers_amd::_layer_norm_backward");
        check_backward(grads[0]);
        const variable_list s = ctx->get_saved_variables();
        Below below;
        auto [dx, dw, db] = back.call(grads[0], s[0], maybe(s[1]), maybe(s[2]), s[3], ctx->saved_data["eps"].toDouble(),
                                      Wanted{ctx->needs_input_grad(0), s[1].defined() && ctx->needs_input_grad(1), s[2].defined() && ctx->needs_input_grad(2)});
        return {dx, dw, db, Tensor(), Tensor()};
    }
};
Tensor layer_norm_autograd(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps)
{
    static const auto plain = op<Tensor(const Tensor&, const MaybeTensor&, const MaybeTensor&, double)>("diffusers_amd::layer_norm");
    no_tangent({x, or_none(weight), or_none(bias)});
    if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias))) {
        leaves_of_this_capture(x, {x, or_none(weight), or_none(bias)});
        return LayerNorm::apply(x, or_x(weight, x), or_x(bias, x), Given{weight.has_value(), bias.has_value()}, eps);
    }
    Below below;
    return plain.call(x, weight, bias, eps);
}

// ------------------------------------------------------------------------------------------ gated feed-forward
struct FfInputs { Tensor x, weight, bias; sde_gated_ff_args a{}; };
FfInputs ff_inputs(const Tensor& x, const Tensor& weight, const MaybeTensor& bias_, int64_t act)
{
    first_tensor(x);
    FfInputs in;
    beside(weight, x, "weight");
    beside(in.bias = or_none(bias_), x, "bias");
    const int64_t step = 16 / x.element_size();
    if (x.dim() == 0 || weight.dim() != 2 || weight.size(1) != x.size(-1) || weight.size(0) % 2)
        bad_value(text("x [..., K] and weight [2F, K], not ", x.sizes(), " and ", weight.sizes()));
    if (weight.scalar_type() != x.scalar_type()) bad_type(text("weight is ", weight.scalar_type(), ", x is ", x.scalar_type()));
    const int64_t k = x.size(-1), f = weight.size(0) / 2;
    if (!k || !f || k % step || f % step) bad_value(text("K and F are positive multiples of ", step, " for ", x.scalar_type()));
    in.bias = param(in.bias, x, 2 * f, "bias");
    in.x = as_rows(x, 16);
    in.weight = as_rows(weight, 16);
    sde_gated_ff_args& a = in.a;
    a.dtype = dtype_of(x);
    a.bias_dtype = in.bias.defined() ? dtype_of(in.bias) : a.dtype;
    a.activation = (int)act;
    a.M = rows_of(x);
    a.K = k;
    a.F = f;
    a.ld_x = ld(in.x);
    a.ld_w = ld(in.weight);
    a.ld_h = f;
    a.ld_dx = a.ld_dw = k;
    if (x.is_meta()) return in;
    a.x = ptr(in.x);
    a.weight = ptr(in.weight);
    a.bias = ptr(in.bias);
    return in;
}
Tensor with_last(const Tensor& x, int64_t n)          // of x's leading shape
{
    c10::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    return at::empty(shape, x.options());
}
Tensor gated_ff(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, int64_t act)
{
    FfInputs in = ff_inputs(x, weight, bias, act);
    Tensor h = with_last(x, in.a.F);
    if (x.is_meta()) return h;
    in.a.h = ptr(h);
    size_t n = 0;
    done(entry.ff_workspace(&in.a, 0, &n));
    Exec ex(x, n);
    done(entry.ff_forward(&in.a, &ex.e));
    return h;
}
std::tuple<Tensor, Tensor, Tensor> gated_ff_backward(const Tensor& dh, const Tensor& x, const Tensor& weight, const MaybeTensor& bias, int64_t act, Wanted wanted)
{
    FfInputs in = ff_inputs(x, weight, bias, act);
    sde_gated_ff_args& a = in.a;
    Tensor dx, dw, db;
    if (wanted[0]) dx = at::empty(x.sizes(), x.options());
    if (wanted[1]) dw = at::empty(weight.sizes(), weight.options());
    if (wanted[2]) db = at::empty(in.bias.sizes(), in.bias.options());
    if (x.is_meta()) return {dx, dw, db};
    const Tensor d2 = as_rows(dh, 16);
    a.ld_dh = ld(d2);
    a.dh = ptr(d2);
    a.dx = ptr(dx);
    a.dweight = ptr(dw);
    a.dbias = ptr(db);
    size_t n = 0;
    done(entry.ff_workspace(&a, 1, &n));
    Exec ex(x, n);
    done(entry.ff_backward(&a, &ex.e));
    return {dx, dw, db};
}
struct GatedFf : torch::autograd::Function<GatedFf> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& weight_, const Tensor& b, Given given, int64_t act)
    {
        static const auto plain = op<Tensor(const Tensor&, const Tensor&, const MaybeTensor&, int64_t)>("diffusers_amd::gated_ff");
        Below below;
        const bool rows = x_.dim() && weight_.dim();
        const Tensor x = rows ? as_rows(x_, 16) : x_, weight = rows ? as_rows(weight_, 16) : weight_, bias = given.bias ? b : Tensor();
        Tensor h = plain.call(x, weight, maybe(bias), act);
        ctx->save_for_backward({x, weight, bias});
        ctx->saved_data["act"] = act;
        return h;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        static const auto back = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, int64_t, Wanted)>("diffusers_amd::_gated_ff_backward");
        check_backward(grads[0]);
        const variable_list s = ctx->get_saved_variables();
        Below below;
        auto [dx, dw, db] = back.call(grads[0], s[0], s[1], maybe(s[2]), ctx->saved_data["act"].toInt(),
                                      Wanted{ctx->needs_input_grad(0), ctx->needs_input_grad(1), s[2].defined() && ctx->needs_input_grad(2)});
        return {dx, dw, db, Tensor(), Tensor()};
    }
};
Tensor gated_ff_autograd(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, int64_t act)
{
    static const auto plain = op<Tensor(const Tensor&, const Tensor&, const MaybeTensor&, int64_t)>("diffusers_amd::gated_ff");
    no_tangent({x, weight, or_none(bias)});
    if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias))) {
        leaves_of_this_capture(x, {x, weight, or_none(bias)});
        return GatedFf::apply(x, weight, or_x(bias, x), Given{true, bias.has_value()}, act);
    }
    Below below;
    return plain.call(x, weight, bias, act);
}

// ------------------------------------------------------------------------------------------ cross attention
// x [B, S, H, D] as the kernels take it: last axis contiguous, every (b, s, h) on 16 bytes, offsets inside a tile within 2 GB
Tensor as_heads(const Tensor& x)
{
    const int64_t e = x.element_size(), step = 16 / e;
    if (x.stride(3) != 1 || x.stride(0) % step || x.stride(1) % step || x.stride(2) % step || !aligned(x, 16) ||
        (65 * x.stride(1) + x.size(2) * x.stride(2) + x.size(3)) * e >= (int64_t(1) << 31))
        return x.clone(at::MemoryFormat::Contiguous);
    return x;
}
// int32, contiguous
Tensor lengths(const Tensor& t, int64_t b, const char* name)
{
    if (!t.defined()) return t;
    if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.dim() != 1 || t.size(0) != b)
        bad_value(text(name, " is an int32 (or int64) tensor of shape [", b, "]"));
    return (t.scalar_type() == at::kLong ? t.clamp(0, INT32_MAX).to(at::kInt) : t).contiguous();
}
void strides(int64_t (&s)[3], const Tensor& t)
{
    if (t.defined())
        for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}
struct XaInputs { Tensor q, k, v, q_lens, kv_lens, mask; double scale; };
// checked, and laid out as the kernels take them
XaInputs xa_inputs(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& q_lens_, const MaybeTensor& kv_lens_, const MaybeTensor& mask_, std::optional<double> scale_)
{
    first_tensor(q);
    XaInputs in;
    beside(k, q, "k");
    beside(v, q, "v");
    beside(in.q_lens = or_none(q_lens_), q, "q_lens");
    beside(in.kv_lens = or_none(kv_lens_), q, "kv_lens");
    beside(in.mask = or_none(mask_), q, "key_mask");
    if (q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
        bad_value(text("q [B, Sq, H, D] and k, v [B, Skv, Hkv, D], not ", q.sizes(), ", ", k.sizes(), ", ", v.sizes()));
    if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) bad_type("q, k and v have one type");
    const int64_t b = q.size(0), h = q.size(2), d = q.size(3), hk = k.size(2), skv = k.size(1), step = 16 / q.element_size();
    if (!h || !hk || h % hk || d <= 0 || d > 256 || d % step)
        bad_value(text("H is a multiple of Hkv, and D at most 256 and a multiple of ", step, " for ", q.scalar_type()));
    in.scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)d);
    if (!(in.scale > 0.0) || !std::isfinite((float)in.scale * 1.5f)) bad_value("scale is positive and finite");
    in.q_lens = lengths(in.q_lens, b, "q_lens");
    in.kv_lens = lengths(in.kv_lens, b, "kv_lens");
    Tensor& mask = in.mask;
    if (mask.defined()) {
        if ((mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte) || mask.dim() != 2 || mask.size(0) != b || mask.size(1) != skv)
            bad_value(text("key_mask is a bool tensor of shape [", b, ", ", skv, "]"));
        if ((skv > 1 && mask.stride(1) != 1) || (b > 1 && mask.stride(0) < skv)) mask = mask.contiguous();
    }
    in.q = as_heads(q);
    in.k = as_heads(k);
    in.v = as_heads(v);
    return in;
}
sde_cross_attention_args xa_args(const XaInputs& in, const Tensor& o, const Tensor& lse)
{
    sde_cross_attention_args a{};
    a.dtype = dtype_of(in.q);
    a.B = in.q.size(0);
    a.Sq = in.q.size(1);
    a.H = in.q.size(2);
    a.D = in.q.size(3);
    a.Skv = in.k.size(1);
    a.Hkv = in.k.size(2);
    a.scale = (float)in.scale;
    a.q = ptr(in.q);
    a.k = ptr(in.k);
    a.v = ptr(in.v);
    a.o = ptr(o);
    a.lse = (float*)ptr(lse);
    a.q_lens = (const int32_t*)ptr(in.q_lens);
    a.kv_lens = (const int32_t*)ptr(in.kv_lens);
    a.key_mask = (const uint8_t*)ptr(in.mask);
    a.key_mask_stride = in.mask.defined() ? in.mask.stride(0) : 0;
    strides(a.q_stride, in.q);
    strides(a.k_stride, in.k);
    strides(a.v_stride, in.v);
    strides(a.o_stride, o);
    return a;
}
Tensor xa_forward(const XaInputs& in, Tensor* lse)
{
    const Tensor& q = in.q;
    Tensor o = at::empty(q.sizes(), q.options());
    if (lse) *lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    if (q.is_meta()) return o;
    sde_cross_attention_args a = xa_args(in, o, lse ? *lse : Tensor());
    size_t n = 0;
    done(entry.xa_workspace(&a, 0, &n));
    Exec ex(q, n);
    done(entry.xa_forward(&a, &ex.e));
    return o;
}
Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& q_lens, const MaybeTensor& kv_lens, const MaybeTensor& mask, std::optional<double> scale)
{
    return xa_forward(xa_inputs(q, k, v, q_lens, kv_lens, mask, scale), nullptr);
}
std::tuple<Tensor, Tensor> cross_attention_kept(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& q_lens, const MaybeTensor& kv_lens, const MaybeTensor& mask, double scale)
{
    Tensor lse, o = xa_forward(xa_inputs(q, k, v, q_lens, kv_lens, mask, scale), &lse);
    return {o, lse};
}
std::tuple<Tensor, Tensor, Tensor> cross_attention_backward(const Tensor& d_o_, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const MaybeTensor& q_lens,
                                                            const MaybeTensor& kv_lens, const MaybeTensor& mask, double scale, Wanted wanted)
{
    const XaInputs in = xa_inputs(q, k, v, q_lens, kv_lens, mask, scale);
    Tensor dq, dk, dv;
    if (wanted[0]) dq = at::empty(q.sizes(), q.options());
    if (wanted[1]) dk = at::empty(k.sizes(), k.options());
    if (wanted[2]) dv = at::empty(v.sizes(), v.options());
    if (q.is_meta()) return {dq, dk, dv};
    const Tensor d_o = as_heads(d_o_);
    sde_cross_attention_args a = xa_args(in, o, lse);
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
    return {dq, dk, dv};
}
struct Counts { MaybeTensor q_lens, kv_lens, mask; };      // no gradients
struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Counts& n, std::optional<double> scale)
    {
        static const auto kept = op<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&, double)>(
            "diffusers_amd::_cross_attention_kept");
        Below below;
        const XaInputs in = xa_inputs(q, k, v, n.q_lens, n.kv_lens, n.mask, scale);        // kept as they were laid out: the backward pass copies nothing again
        auto [o, lse] = kept.call(in.q, in.k, in.v, maybe(in.q_lens), maybe(in.kv_lens), maybe(in.mask), in.scale);
        ctx->save_for_backward({in.q, in.k, in.v, o, lse, in.q_lens, in.kv_lens, in.mask});
        ctx->saved_data["scale"] = in.scale;
        return o;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        static const auto back = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&,
                                                                       const MaybeTensor&, const MaybeTensor&, double, Wanted)>("diffusers_amd::_cross_attention_backward");
        check_backward(grads[0]);
        const variable_list s = ctx->get_saved_variables();
        Below below;
        auto [dq, dk, dv] = back.call(grads[0], s[0], s[1], s[2], s[3], s[4], maybe(s[5]), maybe(s[6]), maybe(s[7]), ctx->saved_data["scale"].toDouble(),
                                      Wanted{ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)});
        return {dq, dk, dv, Tensor(), Tensor()};
    }
};
Tensor cross_attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& q_lens, const MaybeTensor& kv_lens, const MaybeTensor& mask, std::optional<double> scale)
{
    static const auto plain = op<Tensor(const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&, std::optional<double>)>(
        "diffusers_amd::cross_attention");
    no_tangent({q, k, v});
    if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v))) {
        leaves_of_this_capture(q, {q, k, v});
        return CrossAttention::apply(q, k, v, Counts{q_lens, kv_lens, mask}, scale);
    }
    Below below;
    return plain.call(q, k, v, q_lens, kv_lens, mask, scale);
}

// the CUDA and the Meta entries: the same functions, which launch nothing for tensors without memory
void entries(torch::Library& m)
{
    m.impl("layer_norm", &layer_norm);
    m.impl("_layer_norm_kept", &layer_norm_kept);
    m.impl("_layer_norm_backward", &layer_norm_backward);
    m.impl("gated_ff", &gated_ff);
    m.impl("_gated_ff_backward", &gated_ff_backward);
    m.impl("cross_attention", &cross_attention);
    m.impl("_cross_attention_kept", &cross_attention_kept);
    m.impl("_cross_attention_backward", &cross_attention_backward);
}

// What diffusers_amd.ops calls.  torch.jit's tracer records calls that come through torch.ops alone; all others go straight to the dispatcher.
template <typename F, typename... A> Tensor call(const char* name, const c10::TypedOperatorHandle<F>& handle, const Tensor& first, const A&... rest)
{
    on_a_gpu(first);
    if (torch::jit::tracer::isTracing()) return py::module_::import("torch").attr("ops").attr("diffusers_amd").attr(name)(first, rest...).template cast<Tensor>();
    return handle.call(first, rest...);
}

}  // namespace

TORCH_LIBRARY(diffusers_amd, m)
{
    m.def("layer_norm(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> Tensor");
    m.def("_layer_norm_kept(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
    m.def("_layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, float eps, bool[3] wanted) -> (Tensor, Tensor, Tensor)");
    m.def("gated_ff(Tensor x, Tensor weight, Tensor? bias=None, int activation=0) -> Tensor");
    m.def("_gated_ff_backward(Tensor dh, Tensor x, Tensor weight, Tensor? bias, int activation, bool[3] wanted) -> (Tensor, Tensor, Tensor)");
    m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? q_lens=None, Tensor? kv_lens=None, Tensor? key_mask=None, float? scale=None) -> Tensor");
    m.def("_cross_attention_kept(Tensor q, Tensor k, Tensor v, Tensor? q_lens, Tensor? kv_lens, Tensor? key_mask, float scale) -> (Tensor, Tensor)");
    m.def("_cross_attention_backward(Tensor d_o, Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor? q_lens, Tensor? kv_lens, Tensor? key_mask, float scale, bool[3] wanted) -> "
          "(Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(diffusers_amd, CUDA, m) { entries(m); }
TORCH_LIBRARY_IMPL(diffusers_amd, Meta, m) { entries(m); }
TORCH_LIBRARY_IMPL(diffusers_amd, Autograd, m)
{
    m.impl("layer_norm", &layer_norm_autograd);
    m.impl("gated_ff", &gated_ff_autograd);
    m.impl("cross_attention", &cross_attention_autograd);
}

PYBIND11_MODULE(_torch_ops, m)
{
    m.def("bind", [](const py::dict& at, py::object error) {
        auto take = [&](auto& f, const char* name) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at[name].cast<uintptr_t>()); };
        take(entry.ln_forward, "sde_layer_norm_forward");
        take(entry.ln_backward, "sde_layer_norm_backward");
        take(entry.ln_workspace, "sde_layer_norm_workspace");
        take(entry.ff_forward, "sde_gated_ff_forward");
        take(entry.ff_backward, "sde_gated_ff_backward");
        take(entry.ff_workspace, "sde_gated_ff_workspace");
        take(entry.xa_forward, "sde_cross_attention_forward");
        take(entry.xa_backward, "sde_cross_attention_backward");
        take(entry.xa_workspace, "sde_cross_attention_workspace");
        if (!sde_error) sde_error = error.release().ptr();
        take(entry.last_error, "sde_last_error");                // last: it marks the rest as there
    });
    m.def("layer_norm", torch::wrap_pybind_function([](const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
        static const auto handle = op<Tensor(const Tensor&, const MaybeTensor&, const MaybeTensor&, double)>("diffusers_amd::layer_norm");
        return call("layer_norm", handle, x, weight, bias, eps);
    }));
    m.def("gated_ff", torch::wrap_pybind_function([](const Tensor& x, const Tensor& weight, const MaybeTensor& bias, int64_t act) {
        static const auto handle = op<Tensor(const Tensor&, const Tensor&, const MaybeTensor&, int64_t)>("diffusers_amd::gated_ff");
        return call("gated_ff", handle, x, weight, bias, act);
    }));
    m.def("cross_attention", torch::wrap_pybind_function([](const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& q_lens, const MaybeTensor& kv_lens,
                                                            const MaybeTensor& mask, std::optional<double> scale) {
        static const auto handle = op<Tensor(const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&, std::optional<double>)>(
            "diffusers_amd::cross_attention");
        return call("cross_attention", handle, q, k, v, q_lens, kv_lens, mask, scale);
    }));
}
