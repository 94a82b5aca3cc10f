// Matrix products with an epilogue and their backward pass: the entry points and what they refuse (the kernels: skm_linear_kernels.h).
#include "skm_linear.h"

namespace {

int check_matrix(const char *who, const char *what, const void *p, int64_t rows, int64_t cols, int64_t ld, int64_t es)
{
    SKM_REQUIRE(ld >= cols, SKM_E_BADARG, "%s: the row stride of %s (%lld) is less than its %lld columns", who, what, (long long)ld, (long long)cols);
    SKM_REQUIRE((uintptr_t)p % (uintptr_t)es == 0, SKM_E_BADARG, "%s: %s is not aligned to its type", who, what);
    return SKM_OK;
}

}  // namespace

extern "C" int skm_linear(skm_ctx *ctx, int dtype, int activation, int64_t m, int64_t n, int64_t k, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw,
                          const void *d_bias, const void *d_residual, int64_t ldr, void *d_preact, int64_t ldp, void *d_y, int64_t ldy)
{
    const char *who = "skm_linear";
    SKM_REQUIRE(ctx, SKM_E_BADARG, "%s: null context", who);
    SKM_REQUIRE(dtype >= 0 && dtype <= 2, SKM_E_BADARG, "%s: dtype must be 0 (float32), 1 (float16) or 2 (bfloat16)", who);
    SKM_REQUIRE(activation >= 0 && activation < ACT_COUNT, SKM_E_BADARG, "%s: unknown activation %d", who, activation);
    SKM_REQUIRE(m >= 0 && n >= 0 && k >= 0, SKM_E_BADARG, "%s: negative size", who);
    if (m == 0 || n == 0)
        return SKM_OK;
    const int64_t es = (int64_t)elem_bytes(dtype);
    SKM_REQUIRE(d_y && (k == 0 || (d_x && d_w)), SKM_E_BADARG, "%s: null array", who);
    SKM_TRY(check_matrix(who, "x", d_x, m, k, ldx, es));
    SKM_TRY(check_matrix(who, "w", d_w, n, k, ldw, es));
    SKM_TRY(check_matrix(who, "y", d_y, m, n, ldy, es));
    SKM_REQUIRE((uintptr_t)d_bias % (uintptr_t)es == 0, SKM_E_BADARG, "%s: bias is not aligned to its type", who);
    if (d_residual)
        SKM_TRY(check_matrix(who, "residual", d_residual, m, n, ldr, es));
    if (d_preact)
        SKM_TRY(check_matrix(who, "preact", d_preact, m, n, ldp, es));
    void *const outs[2] = {d_y, d_preact};
    const int64_t ldos[2] = {ldy, ldp};
    for (int o = 0; o < 2; ++o) {
        SKM_REQUIRE(!skm_overlap(outs[o], m, n, ldos[o], d_x, m, k, ldx, es) && !skm_overlap(outs[o], m, n, ldos[o], d_w, n, k, ldw, es) &&
                        !skm_overlap(outs[o], m, n, ldos[o], d_bias, 1, n, n, es),
                    SKM_E_BADARG, "%s: an output shares memory with x, w or bias", who);
        // (a cell of the residual is read by the lane that writes that cell: the output may BE the residual)
        SKM_REQUIRE((outs[o] == d_residual && ldos[o] == ldr && o == 0) || !skm_overlap(outs[o], m, n, ldos[o], d_residual, m, n, ldr, es), SKM_E_BADARG,
                    "%s: an output shares memory with the residual without being it", who);
    }
    SKM_REQUIRE(!skm_overlap(d_y, m, n, ldy, d_preact, m, n, ldp, es), SKM_E_BADARG, "%s: y and preact share memory", who);
    SKM_ON_DEVICE(ctx);
    if (dtype == 0)
        return skm_linear_forward<0>(ctx, activation, m, n, k, d_x, ldx, d_w, ldw, d_bias, d_residual, ldr, d_preact, ldp, d_y, ldy);
    if (dtype == 1)
        return skm_linear_forward<1>(ctx, activation, m, n, k, d_x, ldx, d_w, ldw, d_bias, d_residual, ldr, d_preact, ldp, d_y, ldy);
    return skm_linear_forward<2>(ctx, activation, m, n, k, d_x, ldx, d_w, ldw, d_bias, d_residual, ldr, d_preact, ldp, d_y, ldy);
}

extern "C" int skm_linear_backward(skm_ctx *ctx, int dtype, int activation, int64_t m, int64_t n, int64_t k, const void *d_dy, int64_t lddy, const void *d_preact,
                                   int64_t ldp, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, void *d_dx, int64_t lddx, void *d_dw, int64_t lddw,
                                   void *d_dbias)
{
    const char *who = "skm_linear_backward";
    SKM_REQUIRE(ctx, SKM_E_BADARG, "%s: null context", who);
    SKM_REQUIRE(dtype >= 0 && dtype <= 2, SKM_E_BADARG, "%s: dtype must be 0 (float32), 1 (float16) or 2 (bfloat16)", who);
    SKM_REQUIRE(activation >= 0 && activation < ACT_COUNT, SKM_E_BADARG, "%s: unknown activation %d", who, activation);
    SKM_REQUIRE(m >= 0 && n >= 0 && k >= 0, SKM_E_BADARG, "%s: negative size", who);
    // (a gradient without cells may have no address)
    SKM_REQUIRE(d_dx || d_dw || d_dbias || m == 0 || n == 0 || k == 0, SKM_E_BADARG, "%s: no gradient is asked for", who);
    const int64_t es = (int64_t)elem_bytes(dtype);
    const bool cells = m > 0 && n > 0;
    SKM_REQUIRE(!cells || d_dy, SKM_E_BADARG, "%s: null dy", who);
    SKM_REQUIRE(!cells || activation == ACT_NONE || d_preact, SKM_E_BADARG, "%s: the activation's slope needs the pre-activation values", who);
    SKM_REQUIRE(!d_dx || n == 0 || k == 0 || d_w, SKM_E_BADARG, "%s: dx needs w", who);
    SKM_REQUIRE(!d_dw || m == 0 || k == 0 || d_x, SKM_E_BADARG, "%s: dw needs x", who);
    if (cells)
        SKM_TRY(check_matrix(who, "dy", d_dy, m, n, lddy, es));
    if (cells && activation != ACT_NONE)
        SKM_TRY(check_matrix(who, "preact", d_preact, m, n, ldp, es));
    if (d_dx) {
        SKM_TRY(check_matrix(who, "w", d_w, n, k, ldw, es));
        SKM_TRY(check_matrix(who, "dx", d_dx, m, k, lddx, es));
    }
    if (d_dw) {
        SKM_TRY(check_matrix(who, "x", d_x, m, k, ldx, es));
        SKM_TRY(check_matrix(who, "dw", d_dw, n, k, lddw, es));
    }
    SKM_REQUIRE((uintptr_t)d_dbias % (uintptr_t)es == 0, SKM_E_BADARG, "%s: dbias is not aligned to its type", who);
    struct part {
        const void *p;
        int64_t rows, cols, ld;
    };
    const part in[4] = {{d_dy, m, n, lddy}, {activation != ACT_NONE ? d_preact : nullptr, m, n, ldp}, {d_dw ? d_x : nullptr, m, k, ldx}, {d_dx ? d_w : nullptr, n, k, ldw}};
    const part out[3] = {{d_dx, m, k, lddx}, {d_dw, n, k, lddw}, {d_dbias, 1, n, n}};
    for (int o = 0; o < 3; ++o) {
        for (const part &i : in)
            SKM_REQUIRE(!skm_overlap(out[o].p, out[o].rows, out[o].cols, out[o].ld, i.p, i.rows, i.cols, i.ld, es), SKM_E_BADARG, "%s: a gradient shares memory with an input", who);
        for (int q = 0; q < o; ++q)
            SKM_REQUIRE(!skm_overlap(out[o].p, out[o].rows, out[o].cols, out[o].ld, out[q].p, out[q].rows, out[q].cols, out[q].ld, es), SKM_E_BADARG,
                        "%s: two gradients share memory", who);
    }
    SKM_ON_DEVICE(ctx);
    // (k = 0: dx and dw have no cells, the bias's gradient is what is left; m or n = 0: what has cells is an empty sum)
    void *dx = m && k ? d_dx : nullptr, *dw = n && k ? d_dw : nullptr, *db = n ? d_dbias : nullptr;
    if (!dx && !dw && !db)
        return SKM_OK;
    if (dtype == 0)
        return skm_linear_gradients<0>(ctx, activation, m, n, k, d_dy, lddy, d_preact, ldp, d_x, ldx, d_w, ldw, dx, lddx, dw, lddw, db);
    if (dtype == 1)
        return skm_linear_gradients<1>(ctx, activation, m, n, k, d_dy, lddy, d_preact, ldp, d_x, ldx, d_w, ldw, dx, lddx, dw, lddw, db);
    return skm_linear_gradients<2>(ctx, activation, m, n, k, d_dy, lddy, d_preact, ldp, d_x, ldx, d_w, ldw, dx, lddx, dw, lddw, db);
}
