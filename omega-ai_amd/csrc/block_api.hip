// C entries of the operators around the experts of a block: RMS norm with the residual's addition, rows kept in 8 bits.
// Everything that can be checked without the device is checked here; the launchers get arguments they can trust.
#include <math.h>

#include "ops_check.h"

static bool form_ok(int form) { return form == OMEGA_KEEP8_INT8 || form == OMEGA_KEEP8_MX; }
// bytes of the scales of [T,d] and of one scale
static size_t scale_bytes(int form, int T, int d) { return (size_t)T * (form == OMEGA_KEEP8_MX ? (size_t)ceil_div(d, 32) : (size_t)ceil_div(d, 128) * 4); }

extern "C" {

int omega_hip_rmsnorm_forward(omega_ctx *ctx, const void *x, const void *residual, int dtype, int T, int d, const float *gamma, float eps, void *sum,
                              void *out, uint8_t *out8, uint8_t *out8_scales, uint8_t *keep8, float *keep8_scales, float *rstd)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, 1, d)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_forward: bad dtype or size");
    if (!(eps >= 0.0f) || isinf(eps)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_forward: eps must be finite and not negative");
    if (T == 0) return OMEGA_OK;
    if (!x || !gamma || (!out && !out8)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_forward: NULL pointer");
    if ((out8 != nullptr) != (out8_scales != nullptr) || (keep8 != nullptr) != (keep8_scales != nullptr))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_forward: codes without scales, or scales without codes");
    if (sum && !residual) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_forward: a sum without a residual");
    const size_t es = dtype_size(dtype), e = (size_t)T * d, n = e * es, T4 = (size_t)T * 4, d4 = (size_t)d * 4;
    if (misaligned(x, es) || misaligned(residual, es) || misaligned(sum, es) || misaligned(out, es) || misaligned(gamma, 4) || misaligned(keep8_scales, 4) ||
        misaligned(rstd, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_forward: misaligned pointer");
    // (the sum in place: it is that input's span)
    const bool on_x = sum && sum == x, on_res = sum && sum == residual;
    span s[] = {on_x ? out_span(x, n) : in_span(x, n), on_res ? out_span(residual, n) : in_span(residual, residual ? n : 0), in_span(gamma, d4),
                out_span(sum, sum && !on_x && !on_res ? n : 0), out_span(out, out ? n : 0), out_span(out8, out8 ? e : 0),
                out_span(out8_scales, out8 ? scale_bytes(OMEGA_KEEP8_MX, T, d) : 0), out_span(keep8, keep8 ? e : 0),
                out_span(keep8_scales, keep8 ? scale_bytes(OMEGA_KEEP8_INT8, T, d) : 0), out_span(rstd, rstd ? T4 : 0)};
    if (overlapping(s, 10)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_forward: buffers overlap");
    const rmsnorm_forward a = {x, residual, dtype, T, d, gamma, eps, sum, out, out8, out8_scales, keep8, keep8_scales, rstd};
    OMEGA_HIP_CHECK(ctx, launch_rmsnorm_forward(ctx, a, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_rmsnorm_backward(omega_ctx *ctx, const void *h, const uint8_t *keep8, const float *keep8_scales, const void *dout, const void *dsum, int dtype,
                               int T, int d, const float *gamma, const float *rstd, void *dx, float *dgamma)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, 1, d)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_backward: bad dtype or size");
    if (!dgamma || (T > 0 && (!dout || !gamma || !rstd || !dx))) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_backward: NULL pointer");
    if (T > 0 && ((h != nullptr) == (keep8 != nullptr) || (keep8 != nullptr) != (keep8_scales != nullptr)))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_backward: the input is either rows or codes with their scales");
    const size_t es = dtype_size(dtype), e = (size_t)T * d, n = e * es, T4 = (size_t)T * 4, d4 = (size_t)d * 4;
    if (misaligned(h, es) || misaligned(dout, es) || misaligned(dsum, es) || misaligned(dx, es) || misaligned(gamma, 4) || misaligned(rstd, 4) ||
        misaligned(dgamma, 4) || misaligned(keep8_scales, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_backward: misaligned pointer");
    const bool on_dsum = dsum && dx == dsum;
    span s[] = {in_span(h, h ? n : 0), in_span(keep8, keep8 ? e : 0), in_span(keep8_scales, keep8 ? scale_bytes(OMEGA_KEEP8_INT8, T, d) : 0), in_span(dout, n),
                in_span(dsum, dsum && !on_dsum ? n : 0), in_span(gamma, T ? d4 : 0), in_span(rstd, T4), out_span(dx, n), out_span(dgamma, d4)};
    if (overlapping(s, 9)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "rmsnorm_backward: buffers overlap");
    void *ws;
    WORKSPACE(ctx, rmsnorm_backward_workspace(ctx, T, d), &ws);
    const rmsnorm_backward a = {h, keep8, keep8_scales, dout, dsum, dtype, T, d, gamma, rstd, dx, dgamma};
    OMEGA_HIP_CHECK(ctx, launch_rmsnorm_backward(ctx, a, ws, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_keep8_save(omega_ctx *ctx, const void *x, int dtype, int T, int d, int form, uint8_t *codes, void *scales)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, 1, d) || !form_ok(form)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_save: bad dtype, size or form");
    if (T == 0) return OMEGA_OK;
    if (!x || !codes || !scales) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_save: NULL pointer");
    const size_t es = dtype_size(dtype), e = (size_t)T * d;
    if (misaligned(x, es) || (form == OMEGA_KEEP8_INT8 && misaligned(scales, 4))) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_save: misaligned pointer");
    span s[] = {in_span(x, e * es), out_span(codes, e), out_span(scales, scale_bytes(form, T, d))};
    if (overlapping(s, 3)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_save: buffers overlap");
    OMEGA_HIP_CHECK(ctx, launch_keep8_save(x, dtype, T, d, form, codes, scales, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_keep8_load(omega_ctx *ctx, const uint8_t *codes, const void *scales, int form, int T, int d, void *out, int dtype)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, 1, d) || !form_ok(form)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_load: bad dtype, size or form");
    if (T == 0) return OMEGA_OK;
    if (!codes || !scales || !out) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_load: NULL pointer");
    const size_t es = dtype_size(dtype), e = (size_t)T * d;
    if (misaligned(out, es) || (form == OMEGA_KEEP8_INT8 && misaligned(scales, 4))) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_load: misaligned pointer");
    span s[] = {in_span(codes, e), in_span(scales, scale_bytes(form, T, d)), out_span(out, e * es)};
    if (overlapping(s, 3)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "keep8_load: out overlaps an input");
    OMEGA_HIP_CHECK(ctx, launch_keep8_load(codes, scales, form, T, d, out, dtype, ctx->stream));
    return OMEGA_OK;
}

}  // extern "C"
