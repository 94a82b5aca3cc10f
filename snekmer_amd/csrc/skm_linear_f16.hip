#include "skm_linear_kernels.h"

template int skm_linear_forward<1>(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *x, int64_t ldx, const void *w, int64_t ldw,
    const void *bias, const void *residual, int64_t ldr, void *preact, int64_t ldp, void *y, int64_t ldy);
template int skm_linear_gradients<1>(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *dy, int64_t lddy, const void *z, int64_t ldz,
    const void *x, int64_t ldx, const void *w, int64_t ldw, void *dx, int64_t lddx, void *dw, int64_t lddw, void *dbias);
