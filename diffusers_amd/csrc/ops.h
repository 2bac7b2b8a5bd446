// ops.h — internal interface of the operators that are callable on their own (layer norm, gated feed-forward, cross attention).
// ops.cpp checks the arguments of the C ABI and lays out the workspace; the launchers below assume checked arguments.
#pragma once
#include "common.h"

struct OpCtx {
    hipStream_t stream;
    char* ws;          // workspace, 256-byte aligned, at least what the matching *_ws_bytes says
};

size_t op_layer_norm_ws_bytes(const sde_layer_norm_args& a);                       // backward; the forward pass needs none
void op_layer_norm_forward(const OpCtx& c, const sde_layer_norm_args& a);
void op_layer_norm_backward(const OpCtx& c, const sde_layer_norm_args& a);

size_t op_gated_ff_ws_bytes(const sde_gated_ff_args& a, bool backward);
void op_gated_ff_forward(const OpCtx& c, const sde_gated_ff_args& a);
void op_gated_ff_backward(const OpCtx& c, const sde_gated_ff_args& a);
struct GffPlan { int cfg, splits; };                                               // tile (0 = 256 x 256, 1 = 128 x 128, 2 = 64 x 64) and parts of the contraction
GffPlan op_gated_ff_plan(const sde_gated_ff_args& a, int product, int64_t* units);  // product: 0 = x W^T, 1 = dx, 2 = dW; units: tiles times parts

size_t op_cross_attention_ws_bytes(const sde_cross_attention_args& a, bool backward);
int64_t op_cross_attention_threads(const sde_cross_attention_args& a);             // of the largest launch: HIP takes less than 2^32
void op_cross_attention_forward(const OpCtx& c, const sde_cross_attention_args& a);
void op_cross_attention_backward(const OpCtx& c, const sde_cross_attention_args& a);

static inline size_t op_align(size_t n) { return (n + 255) & ~(size_t)255; }
static inline size_t op_esize(int dtype) { return dtype == SDE_F32 ? 4 : 2; }
void allow_dynamic_lds(const void* kernel, int bytes);                             // gemm.hip: once per device and kernel
static inline void op_allow_lds(const void* kernel, int bytes) { if (bytes > 65536) allow_dynamic_lds(kernel, bytes); }
// every launch is followed by this: a refused launch is an error of the call, not of a later one
static inline void op_launched(const char* what)
{
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) sde_fail(SDE_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e));
}
