// C entries of the operators around the experts of a block: routing to experts, RMS norm with the residual's addition, rows kept in 8 bits.
// Everything that can be checked without the device is checked here; the launchers get arguments they can trust.
#include <math.h>

#include "ops_check.h"

static bool form_ok(int form) { return form == OMEGA_KEEP8_INT8 || form == OMEGA_KEEP8_MX; }
// bytes of the scales of [T,d] and of one scale
static size_t scale_bytes(int form, int T, int d) { return (size_t)T * (form == OMEGA_KEEP8_MX ? (size_t)ceil_div(d, 32) : (size_t)ceil_div(d, 128) * 4); }

static const char *route_config_wrong(const omega_route_config *c)
{
    if (!c) return "no routing configuration";
    if (c->E < 1 || c->E > 512 || c->K < 1 || c->K > 64) return "routing: E is 1..512, K 1..64";
    if (c->score != OMEGA_ROUTE_SOFTMAX && c->score != OMEGA_ROUTE_SIGMOID) return "routing: unknown score";
    if (c->renorm != 0 && c->renorm != 1) return "routing: renorm is 0 or 1";
    if (c->groups < 1 || c->groups > 64 || c->E % c->groups != 0) return "routing: groups are 1..64 and divide E";
    if (c->top_groups < 1 || c->top_groups > c->groups || c->group_best < 1 || c->group_best > 2) return "routing: top_groups is 1..groups, group_best 1 or 2";
    if (c->K > c->top_groups * (c->E / c->groups)) return "routing: K exceeds the experts of the groups that stay";
    if (!(c->scale > 0.0f) || isinf(c->scale)) return "routing: scale must be positive and finite";
    return nullptr;
}
#define ROUTE_CONFIG(ctx, c)                                                             \
    do {                                                                                 \
        const char *const wrong_ = route_config_wrong(c);                                \
        if (wrong_) OMEGA_FAIL((ctx), OMEGA_ERR_INVALID_ARG, wrong_);                    \
    } while (0)

extern "C" {

int omega_hip_route_forward(omega_ctx *ctx, const omega_route_config *cfg, const float *logits, int T, const float *bias, int32_t *ids, float *w, int32_t *counts)
{
    CTX_ENTER(ctx);
    ROUTE_CONFIG(ctx, cfg);
    if (!sizes_ok(T, 1, cfg->E)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_forward: bad size");
    if (T > 0 && (!logits || !ids || !w)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_forward: NULL pointer");
    if (misaligned(logits, 4) || misaligned(bias, 4) || misaligned(ids, 4) || misaligned(w, 4) || misaligned(counts, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_forward: misaligned pointer");
    const size_t e4 = (size_t)cfg->E * 4, k = (size_t)T * cfg->K * 4;
    span s[] = {in_span(logits, (size_t)T * e4), in_span(bias, bias ? e4 : 0), out_span(ids, k), out_span(w, k), out_span(counts, counts ? e4 : 0)};
    if (overlapping(s, 5)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_forward: buffers overlap");
    if (T == 0 && !counts) return OMEGA_OK;
    void *ws;
    WORKSPACE(ctx, route_workspace(ctx, *cfg, T), &ws);
    OMEGA_HIP_CHECK(ctx, launch_route_forward(ctx, *cfg, logits, T, bias, ids, w, counts, ws, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_route_backward(omega_ctx *ctx, const omega_route_config *cfg, const float *logits, int T, const int32_t *ids, const float *w, const float *dw,
                             float *dlogits)
{
    CTX_ENTER(ctx);
    ROUTE_CONFIG(ctx, cfg);
    if (!sizes_ok(T, 1, cfg->E)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_backward: bad size");
    if (T == 0) return OMEGA_OK;
    const bool asks = cfg->score != OMEGA_ROUTE_SOFTMAX || !cfg->renorm;
    if ((asks && !logits) || !ids || !w || !dw || !dlogits) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_backward: NULL pointer");
    if (misaligned(logits, 4) || misaligned(ids, 4) || misaligned(w, 4) || misaligned(dw, 4) || misaligned(dlogits, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_backward: misaligned pointer");
    const size_t e = (size_t)T * cfg->E * 4, k = (size_t)T * cfg->K * 4;
    span s[] = {in_span(logits, logits ? e : 0), in_span(ids, k), in_span(w, k), in_span(dw, k), out_span(dlogits, e)};
    if (overlapping(s, 5)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_backward: buffers overlap");
    OMEGA_HIP_CHECK(ctx, launch_route_backward(*cfg, logits, T, ids, w, dw, dlogits, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_route_balance(omega_ctx *ctx, const int32_t *counts, int E, float rate, float *bias)
{
    CTX_ENTER(ctx);
    if (E < 1 || E > SIZE_MAX_COLS || !counts || !bias) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_balance: NULL pointer or bad size");
    if (!(rate >= 0.0f) || isinf(rate)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_balance: rate must be finite and not negative");
    if (misaligned(counts, 4) || misaligned(bias, 4)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_balance: misaligned pointer");
    span s[] = {in_span(counts, (size_t)E * 4), out_span(bias, (size_t)E * 4)};
    if (overlapping(s, 2)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "route_balance: buffers overlap");
    OMEGA_HIP_CHECK(ctx, launch_route_balance(counts, E, rate, bias, ctx->stream));
    return OMEGA_OK;
}

int omega_moe_set_routing(omega_moe *m, const omega_route_config *cfg, int with_bias)
{
    if (!m) OMEGA_FAIL(nullptr, OMEGA_ERR_INVALID_ARG, "NULL layer");
    omega_ctx *ctx = m->ctx;
    CTX_ENTER(ctx);
    const size_t E4 = (size_t)m->cfg.E * 4;
    if (cfg) {
        ROUTE_CONFIG(ctx, cfg);
        if (cfg->E != m->cfg.E || cfg->K != m->cfg.K) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "set_routing: E and K are not the layer's");
        // what the routing needs, whole or not at all
        float *bias = m->route_bias, *logits = m->route_logits;
        hipError_t e = hipSuccess;
        if (with_bias && !bias) e = hipMalloc((void **)&bias, E4);
        if (e == hipSuccess && !logits && m->T_cap > 0) e = hipMalloc((void **)&logits, (size_t)m->T_cap * E4);
        if (e == hipSuccess && bias && bias != m->route_bias) e = launch_zero_f32(bias, (size_t)m->cfg.E, ctx->stream);
        if (e != hipSuccess) {
            (void)hipGetLastError();  // the next launch would else report it as its own
            if (bias && bias != m->route_bias) (void)hipFree(bias);
            if (logits && logits != m->route_logits) (void)hipFree(logits);
            return omega_set_error(ctx, e == hipErrorOutOfMemory ? OMEGA_ERR_OOM : OMEGA_ERR_HIP, "set_routing: allocation", e, __FILE__, __LINE__);
        }
        m->route_bias = bias;
        m->route_logits = logits;
        m->route = *cfg;
    }
    if (m->route_bias && !(cfg && with_bias)) {
        OMEGA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));  // a launch may still read it
        OMEGA_HIP_CHECK(ctx, hipFree(m->route_bias));
        m->route_bias = nullptr;
    }
    m->own_routing = cfg != nullptr;
    // the routing of the last batch is another's
    m->fwd_T = -1;
    m->fwd_block = false;
    m->rec_valid = false;
    m->routed_T = m->dispatched_T = -1;
    return OMEGA_OK;
}

int omega_moe_balance(omega_moe *m, float rate)
{
    if (!m) OMEGA_FAIL(nullptr, OMEGA_ERR_INVALID_ARG, "NULL layer");
    omega_ctx *ctx = m->ctx;
    CTX_ENTER(ctx);
    if (!(rate >= 0.0f) || isinf(rate)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "balance: rate must be finite and not negative");
    if (!m->route_bias) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "balance: the layer's routing has no bias");
    if (m->dispatched_T < 0) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "balance: no dispatch has run");
    OMEGA_HIP_CHECK(ctx, launch_route_balance(m->counts, m->cfg.E, rate, m->route_bias, ctx->stream));
    return OMEGA_OK;
}

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
