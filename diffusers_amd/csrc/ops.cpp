// ops.cpp — C ABI of the operators that are callable on their own: argument checks, device, workspace.
#include "ops.h"

#include <algorithm>
#include <cmath>

namespace {

void need(bool ok, const char* msg) { SDE_REQUIRE(ok, SDE_ERR_INVALID_ARGUMENT, msg); }
bool is_dtype(int t) { return t == SDE_F16 || t == SDE_BF16 || t == SDE_F32; }
constexpr int64_t kMaxRows = int64_t(1) << 31;

// makes exec's device current and puts back what was
struct OnDevice {
    int before = -1;
    explicit OnDevice(int id)
    {
        HIP_CHECK(hipGetDevice(&before));
        if (id == before) { before = -1; return; }
        HIP_CHECK(hipSetDevice(id));
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};

template <typename F> sde_status run(const sde_op_exec* e, size_t ws_bytes, F&& f)
{
    need(e != nullptr, "exec is null");
    need(e->device_id >= 0, "device_id is negative");
    if (ws_bytes) {
        need(e->workspace != nullptr && ((uintptr_t)e->workspace & 255) == 0, "workspace is null or not 256-byte aligned");
        if (e->workspace_bytes < ws_bytes)
            sde_fail(SDE_ERR_INVALID_ARGUMENT, "workspace holds " + std::to_string(e->workspace_bytes) + " bytes, " + std::to_string(ws_bytes) + " are needed");
    }
    const OnDevice on(e->device_id);
    f(OpCtx{(hipStream_t)e->hip_stream, (char*)e->workspace});
    return SDE_OK;
}

void check(const sde_layer_norm_args* a)
{
    need(a != nullptr, "args is null");
    need(is_dtype(a->dtype), "layer norm: unknown dtype");
    need(a->param_dtype == a->dtype || a->param_dtype == SDE_F32, "layer norm: param_dtype must be dtype or SDE_F32");
    need(a->rows >= 0 && a->rows < kMaxRows, "layer norm: bad number of rows");
    need(a->C > 0 && a->C <= (1 << 24), "layer norm: C must lie between 1 and 2^24");
    need(a->eps >= 0.0f && std::isfinite(a->eps), "layer norm: eps must be finite and not negative");
}
void ln_ld(int64_t rows, int64_t C, int64_t ld, const char* msg) { need(rows <= 1 || ld >= C, msg); }

void check(const sde_gated_ff_args* a)
{
    need(a != nullptr, "args is null");
    need(is_dtype(a->dtype), "gated ff: unknown dtype");
    need(a->bias_dtype == a->dtype || a->bias_dtype == SDE_F32, "gated ff: bias_dtype must be dtype or SDE_F32");
    need(a->activation >= SDE_ACT_GELU && a->activation <= SDE_ACT_SILU, "gated ff: unknown activation");
    need(a->M >= 0 && a->M < kMaxRows, "gated ff: bad M");
    const int v = 16 / (int)op_esize(a->dtype);
    need(a->K > 0 && a->K <= (1 << 22) && a->K % v == 0, "gated ff: K must be a positive multiple of 16 bytes");
    need(a->F > 0 && a->F <= (1 << 22) && a->F % v == 0, "gated ff: F must be a positive multiple of 16 bytes");
    need((a->M + 255) / 256 * ((a->F + 127) / 128) < kMaxRows, "gated ff: M times F is too large");
    need(a->M < kMaxRows - 256, "gated ff: M is too large");          // a whole K-tile past M is still counted in 32 bits
}
// a matrix of the gated feed-forward: aligned, rows that do not overlap, 256 of them inside a 31-bit window
void matrix(const sde_gated_ff_args& a, const void* p, int64_t ld, int64_t cols, const char* what)
{
    const int64_t e = (int64_t)op_esize(a.dtype);
    if (!p || ((uintptr_t)p & 15) || ld < cols || ld * e % 16 || ld * e >= (1 << 23))
        sde_fail(SDE_ERR_INVALID_ARGUMENT, std::string("gated ff: ") + what + " is null, not 16-byte aligned, or its leading dimension does not fit");
}

void check(const sde_cross_attention_args* a)
{
    need(a != nullptr, "args is null");
    need(is_dtype(a->dtype), "cross attention: unknown dtype");
    need(a->B >= 0 && a->Sq >= 0 && a->Skv >= 0 && a->B < kMaxRows && a->Sq < kMaxRows && a->Skv < kMaxRows - 4096, "cross attention: bad B, Sq or Skv");
    need(a->Hkv > 0 && a->H > 0 && a->H < 65536 && a->H % a->Hkv == 0, "cross attention: H must be a multiple of Hkv");
    need(a->D > 0 && a->D <= 256 && a->D % (16 / (int)op_esize(a->dtype)) == 0, "cross attention: D must be at most 256 and a multiple of 16 bytes");
    need(a->scale > 0.0f && std::isfinite(a->scale * 1.5f), "cross attention: scale must be positive and finite");
    need(a->Sq * (a->H / a->Hkv) < kMaxRows - 4096, "cross attention: too many query rows");
    need(a->B * a->Hkv < (1 << 24), "cross attention: B times Hkv is too large");
    need(!a->key_mask || a->B <= 1 || a->key_mask_stride >= a->Skv, "cross attention: key_mask_stride is less than Skv");
    need(op_cross_attention_threads(*a) < (int64_t(1) << 32), "cross attention: too many workgroups");
}
void tensor(const sde_cross_attention_args& a, const void* p, const int64_t* s, int64_t H, const char* what)
{
    const int64_t e = (int64_t)op_esize(a.dtype);
    bool ok = p && ((uintptr_t)p & 15) == 0;
    for (int i = 0; i < 3; ++i) ok = ok && s[i] >= 0 && s[i] < (int64_t(1) << 40) && s[i] * e % 16 == 0;
    ok = ok && (65 * s[1] + H * s[2] + a.D) * e < kMaxRows;
    if (!ok) sde_fail(SDE_ERR_INVALID_ARGUMENT, std::string("cross attention: ") + what + " is null, not 16-byte aligned, or a stride does not fit");
}
// an output's elements must not share memory
void output(const sde_cross_attention_args& a, const void* p, const int64_t* s, int64_t S, int64_t H, const char* what)
{
    tensor(a, p, s, H, what);
    int64_t size[3] = {a.B, S, H}, str[3] = {s[0], s[1], s[2]};
    for (int i = 0; i < 3; ++i)                       // by stride, smallest first
        for (int j = i + 1; j < 3; ++j)
            if (str[j] < str[i]) { std::swap(str[i], str[j]); std::swap(size[i], size[j]); }
    int64_t span = a.D;
    bool ok = true;
    for (int i = 0; i < 3; ++i) {
        if (size[i] <= 1) continue;
        ok = ok && str[i] >= span;
        span = str[i] * (size[i] - 1) + span;
    }
    if (!ok) sde_fail(SDE_ERR_INVALID_ARGUMENT, std::string("cross attention: elements of ") + what + " overlap");
}

}  // namespace

extern "C" {

sde_status sde_layer_norm_workspace(const sde_layer_norm_args* a, size_t* bytes)
{
    return guarded([&] {
        check(a);
        need(bytes != nullptr, "bytes is null");
        *bytes = op_layer_norm_ws_bytes(*a);
    });
}

sde_status sde_layer_norm_forward(const sde_layer_norm_args* a, const sde_op_exec* exec)
{
    return guarded([&] {
        check(a);
        need(a->rows == 0 || (a->x && a->y), "layer norm: x or y is null");
        need((a->mean == nullptr) == (a->rstd == nullptr), "layer norm: mean and rstd go together");
        ln_ld(a->rows, a->C, a->ld_x, "layer norm: ld_x is less than C");
        ln_ld(a->rows, a->C, a->ld_y, "layer norm: ld_y is less than C");
        run(exec, 0, [&](const OpCtx& c) { op_layer_norm_forward(c, *a); });
    });
}

sde_status sde_layer_norm_backward(const sde_layer_norm_args* a, const sde_op_exec* exec)
{
    return guarded([&] {
        check(a);
        need(a->rows == 0 || (a->x && a->dy && a->mean && a->rstd), "layer norm: x, dy, mean or rstd is null");
        need(a->dx || a->dgamma || a->dbeta || !a->rows, "layer norm: no gradient is asked for");
        ln_ld(a->rows, a->C, a->ld_x, "layer norm: ld_x is less than C");
        ln_ld(a->rows, a->C, a->ld_dy, "layer norm: ld_dy is less than C");
        if (a->dx) ln_ld(a->rows, a->C, a->ld_dx, "layer norm: ld_dx is less than C");
        run(exec, op_layer_norm_ws_bytes(*a), [&](const OpCtx& c) { op_layer_norm_backward(c, *a); });
    });
}

sde_status sde_gated_ff_workspace(const sde_gated_ff_args* a, int backward, size_t* bytes)
{
    return guarded([&] {
        check(a);
        need(bytes != nullptr, "bytes is null");
        *bytes = op_gated_ff_ws_bytes(*a, backward != 0);
    });
}

sde_status sde_gated_ff_forward(const sde_gated_ff_args* a, const sde_op_exec* exec)
{
    return guarded([&] {
        check(a);
        if (a->M) {
            matrix(*a, a->x, a->ld_x, a->K, "x");
            matrix(*a, a->weight, a->ld_w, a->K, "weight");
            matrix(*a, a->h, a->ld_h, a->F, "h");
        }
        run(exec, op_gated_ff_ws_bytes(*a, false), [&](const OpCtx& c) { op_gated_ff_forward(c, *a); });
    });
}

sde_status sde_gated_ff_backward(const sde_gated_ff_args* a, const sde_op_exec* exec)
{
    return guarded([&] {
        check(a);
        need(a->dx || a->dweight || a->dbias || !a->M, "gated ff: no gradient is asked for");
        need(a->F < (1 << 21), "gated ff: F is too large for the backward pass");
        if (a->M) {
            matrix(*a, a->x, a->ld_x, a->K, "x");
            matrix(*a, a->weight, a->ld_w, a->K, "weight");
            matrix(*a, a->dh, a->ld_dh, a->F, "dh");
            if (a->dx) matrix(*a, a->dx, a->ld_dx, a->K, "dx");
        }
        if (a->dweight) matrix(*a, a->dweight, a->ld_dw, a->K, "dweight");
        run(exec, op_gated_ff_ws_bytes(*a, true), [&](const OpCtx& c) { op_gated_ff_backward(c, *a); });
    });
}

sde_status sde_test_gated_ff_plan(const sde_gated_ff_args* a, int product, int* tile, int* splits, int64_t* units)
{
    return guarded([&] {
        check(a);
        need(product >= 0 && product <= 2 && a->M > 0 && tile && splits && units, "gated ff plan: bad product, M or output");
        const GffPlan p = op_gated_ff_plan(*a, product, units);
        *tile = p.cfg;
        *splits = p.splits;
    });
}

sde_status sde_cross_attention_workspace(const sde_cross_attention_args* a, int backward, size_t* bytes)
{
    return guarded([&] {
        check(a);
        need(bytes != nullptr, "bytes is null");
        *bytes = op_cross_attention_ws_bytes(*a, backward != 0);
    });
}

sde_status sde_cross_attention_forward(const sde_cross_attention_args* a, const sde_op_exec* exec)
{
    return guarded([&] {
        check(a);
        if (a->B && a->Sq) {
            output(*a, a->o, a->o_stride, a->Sq, a->H, "o");
            if (a->Skv) {
                tensor(*a, a->q, a->q_stride, a->H, "q");
                tensor(*a, a->k, a->k_stride, a->Hkv, "k");
                tensor(*a, a->v, a->v_stride, a->Hkv, "v");
            }
        }
        run(exec, op_cross_attention_ws_bytes(*a, false), [&](const OpCtx& c) { op_cross_attention_forward(c, *a); });
    });
}

sde_status sde_cross_attention_backward(const sde_cross_attention_args* a, const sde_op_exec* exec)
{
    return guarded([&] {
        check(a);
        need(a->dq || a->dk || a->dv || !a->B || !a->Sq || !a->Skv, "cross attention: no gradient is asked for");
        if (a->dq && a->B && a->Sq) output(*a, a->dq, a->dq_stride, a->Sq, a->H, "dq");
        if (a->dk && a->B && a->Skv) output(*a, a->dk, a->dk_stride, a->Skv, a->Hkv, "dk");
        if (a->dv && a->B && a->Skv) output(*a, a->dv, a->dv_stride, a->Skv, a->Hkv, "dv");
        if (a->B && a->Sq && a->Skv) {
            tensor(*a, a->q, a->q_stride, a->H, "q");
            tensor(*a, a->k, a->k_stride, a->Hkv, "k");
            tensor(*a, a->v, a->v_stride, a->Hkv, "v");
            tensor(*a, a->o, a->o_stride, a->H, "o");
            tensor(*a, a->d_o, a->do_stride, a->H, "d_o");
            need(a->lse != nullptr, "cross attention: lse is null");
        }
        run(exec, op_cross_attention_ws_bytes(*a, true), [&](const OpCtx& c) { op_cross_attention_backward(c, *a); });
    });
}

}  // extern "C"
