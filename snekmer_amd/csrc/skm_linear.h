// What skm_linear.hip (the entry points and their checks) calls, for dtype DT: defined in skm_linear_kernels.h, one translation unit a type.
#pragma once
#include "skm_common.h"

enum { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_SIGMOID, ACT_COUNT };  // activations
constexpr size_t elem_bytes(int dtype) { return dtype == 0 ? 4 : 2; }

template <int DT>
int skm_linear_forward(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *x, int64_t ldx, const void *w, int64_t ldw,
    const void *bias, const void *residual, int64_t ldr, void *preact, int64_t ldp, void *y, int64_t ldy);
template <int DT>
int skm_linear_gradients(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *dy, int64_t lddy, const void *z, int64_t ldz,
    const void *x, int64_t ldx, const void *w, int64_t ldw, void *dx, int64_t lddx, void *dw, int64_t lddw, void *dbias);
