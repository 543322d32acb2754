// C entries of the operators on caller-owned buffers: token embedding, layer norm, head with cross entropy, gradient clipping.
// Everything that can be checked without the device is checked here; the launchers get arguments they can trust.
#include <math.h>

#include <new>

#include "ops_check.h"

static int head_setup(omega_ctx *ctx)
{
    if (!ctx->head_ready) OMEGA_HIP_CHECK(ctx, head_init());
    ctx->head_ready = true;
    return OMEGA_OK;
}

extern "C" {

int omega_hip_embedding_forward(omega_ctx *ctx, const void *table, int dtype, int V, int d, const int32_t *ids, int T, float scale,
                                void *out)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, V, d)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_forward: bad dtype or size");
    if (T == 0) return OMEGA_OK;
    if (!table || !ids || !out) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_forward: NULL pointer");
    const size_t es = dtype_size(dtype);
    if (misaligned(table, es) || misaligned(out, es) || misaligned(ids, 4)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_forward: misaligned pointer");
    span s[] = {in_span(table, (size_t)V * d * es), in_span(ids, (size_t)T * 4), out_span(out, (size_t)T * d * es)};
    if (overlapping(s, 3)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_forward: out overlaps an input");
    OMEGA_HIP_CHECK(ctx, launch_embedding_forward(table, dtype, V, d, ids, T, scale, out, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_embedding_backward(omega_ctx *ctx, const int32_t *ids, int T, const void *dout, int dtype, int V, int d, float scale,
                                 int accumulate, void *dtable, int grad_dtype)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !dtype_ok(grad_dtype) || !sizes_ok(T, V, d))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_backward: bad dtype or size");
    if (!dtable || (T > 0 && (!ids || !dout))) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_backward: NULL pointer");
    const size_t es = dtype_size(dtype), gs = dtype_size(grad_dtype);
    if (misaligned(dtable, gs) || misaligned(dout, es) || misaligned(ids, 4)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_backward: misaligned pointer");
    span s[] = {in_span(ids, (size_t)T * 4), in_span(dout, (size_t)T * d * es), out_span(dtable, (size_t)V * d * gs)};
    if (overlapping(s, 3)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "embedding_backward: dtable overlaps an input");
    if (T == 0 && accumulate) return OMEGA_OK;
    void *ws;
    WORKSPACE(ctx, embedding_backward_workspace(V, d, T), &ws);
    OMEGA_HIP_CHECK(ctx, launch_embedding_backward(ids, T, dout, dtype, V, d, scale, accumulate != 0, dtable, grad_dtype, ws, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_layernorm_forward(omega_ctx *ctx, const void *x, int dtype, int T, int d, const float *gamma, const float *beta, float eps,
                                void *out, float *mean, float *rstd)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, 1, d)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_forward: bad dtype or size");
    if (!(eps >= 0.0f) || isinf(eps)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_forward: eps must be finite and not negative");
    if (T == 0) return OMEGA_OK;
    if (!x || !gamma || !beta || !out) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_forward: NULL pointer");
    const size_t es = dtype_size(dtype), n = (size_t)T * d * es, T4 = (size_t)T * 4, d4 = (size_t)d * 4;
    if (misaligned(x, es) || misaligned(out, es) || misaligned(gamma, 4) || misaligned(beta, 4) || misaligned(mean, 4) || misaligned(rstd, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_forward: misaligned pointer");
    span s[] = {in_span(x, n), in_span(gamma, d4), in_span(beta, d4), out_span(out, n), out_span(mean, mean ? T4 : 0), out_span(rstd, rstd ? T4 : 0)};
    if (overlapping(s, 6)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_forward: buffers overlap");
    OMEGA_HIP_CHECK(ctx, launch_layernorm_forward(ctx, x, dtype, T, d, gamma, beta, eps, out, mean, rstd, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_layernorm_backward(omega_ctx *ctx, const void *x, const void *dout, int dtype, int T, int d, const float *gamma,
                                 const float *mean, const float *rstd, void *dx, float *dgamma, float *dbeta)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, 1, d)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_backward: bad dtype or size");
    if (!dgamma || !dbeta || (T > 0 && (!x || !dout || !gamma || !mean || !rstd || !dx)))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_backward: NULL pointer");
    const size_t es = dtype_size(dtype), n = (size_t)T * d * es, T4 = (size_t)T * 4, d4 = (size_t)d * 4;
    if (misaligned(x, es) || misaligned(dout, es) || misaligned(dx, es) || misaligned(gamma, 4) || misaligned(mean, 4) || misaligned(rstd, 4) ||
        misaligned(dgamma, 4) || misaligned(dbeta, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_backward: misaligned pointer");
    span s[] = {in_span(x, n), in_span(dout, n), in_span(gamma, T ? d4 : 0), in_span(mean, T4), in_span(rstd, T4),
                out_span(dx, n), out_span(dgamma, d4), out_span(dbeta, d4)};
    if (overlapping(s, 8)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "layernorm_backward: buffers overlap");
    void *ws;
    WORKSPACE(ctx, layernorm_backward_workspace(ctx, T, d), &ws);
    OMEGA_HIP_CHECK(ctx, launch_layernorm_backward(ctx, x, dout, dtype, T, d, gamma, mean, rstd, dx, dgamma, dbeta, ws, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_head_loss_forward(omega_ctx *ctx, const void *x, const void *w, int dtype, int T, int V, int d, const int32_t *targets,
                                float *loss, float *row_stats, float *mean)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, V, d)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_forward: bad dtype or size");
    if (!mean || !w || (T > 0 && (!x || !targets || !loss))) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_forward: NULL pointer");
    const size_t es = dtype_size(dtype), T4 = (size_t)T * 4;
    if (misaligned(x, es) || misaligned(w, es) || misaligned(targets, 4) || misaligned(loss, 4) || misaligned(row_stats, 4) || misaligned(mean, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_forward: misaligned pointer");
    span s[] = {in_span(x, (size_t)T * d * es), in_span(w, (size_t)V * d * es), in_span(targets, T4), out_span(loss, T4),
                out_span(row_stats, row_stats ? 2 * T4 : 0), out_span(mean, 8)};
    if (overlapping(s, 6)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_forward: buffers overlap");
    const head_args a = {x, w, dtype, T, V, d, targets, loss, row_stats, mean, nullptr, nullptr, nullptr};
    const int st = head_setup(ctx);
    if (st != OMEGA_OK) return st;
    void *ws;
    WORKSPACE(ctx, head_workspace(ctx, a, false), &ws);
    OMEGA_HIP_CHECK(ctx, launch_head_forward(ctx, a, ws, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_head_loss_backward(omega_ctx *ctx, const void *x, const void *w, int dtype, int T, int V, int d, const int32_t *targets,
                                 const float *row_stats, const float *mean, const float *dloss, void *dx, void *dw)
{
    CTX_ENTER(ctx);
    if (!dtype_ok(dtype) || !sizes_ok(T, V, d)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_backward: bad dtype or size");
    if (!w || !mean || (T > 0 && (!x || !targets || !row_stats))) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_backward: NULL pointer");
    const size_t es = dtype_size(dtype), T4 = (size_t)T * 4, nx = (size_t)T * d * es, nw = (size_t)V * d * es;
    if (misaligned(x, es) || misaligned(w, es) || misaligned(dx, es) || misaligned(dw, es) || misaligned(targets, 4) || misaligned(row_stats, 4) ||
        misaligned(mean, 4) || misaligned(dloss, 4))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_backward: misaligned pointer");
    span s[] = {in_span(x, nx), in_span(w, nw), in_span(targets, T4), in_span(row_stats, 2 * T4), in_span(mean, 8), in_span(dloss, dloss ? 4 : 0),
                out_span(dx, dx ? nx : 0), out_span(dw, dw ? nw : 0)};
    if (overlapping(s, 8)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "head_loss_backward: buffers overlap");
    if (!dx && !dw) return OMEGA_OK;
    const head_args a = {x, w, dtype, T, V, d, targets, nullptr, (float *)row_stats, (float *)mean, dloss, dx, dw};
    const int st = head_setup(ctx);
    if (st != OMEGA_OK) return st;
    void *ws;
    WORKSPACE(ctx, head_workspace(ctx, a, true), &ws);
    OMEGA_HIP_CHECK(ctx, launch_head_backward(ctx, a, ws, ctx->stream));
    return OMEGA_OK;
}

int omega_hip_clip_grad_norm(omega_ctx *ctx, const omega_grad_tensor *tensors, int n_tensors, omega_moe *const *layers, int n_layers,
                             float max_norm, float *norm_out)
{
    CTX_ENTER(ctx);
    if (n_tensors < 0 || n_layers < 0 || (n_tensors > 0 && !tensors) || (n_layers > 0 && !layers))
        OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: bad list of tensors or layers");
    if (!(max_norm >= 0.0f)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: max_norm must not be negative");
    if (misaligned(norm_out, 4)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: misaligned pointer");
    const int n = n_tensors + n_layers;
    // (two spans a tensor at most, and the norm's)
    omega_grad_tensor *all = new (std::nothrow) omega_grad_tensor[(size_t)n + 1];
    span *s = new (std::nothrow) span[2 * (size_t)n + 1];
    struct owner {
        omega_grad_tensor *a;
        span *b;
        ~owner() { delete[] a; delete[] b; }
    } own{all, s};
    if (!all || !s) OMEGA_FAIL(ctx, OMEGA_ERR_OOM, "clip_grad_norm: host allocation failed");
    int m = 0, k = 0;
    auto add = [&](const omega_grad_tensor &t) {
        const size_t bytes = t.n * dtype_size(t.dtype);
        all[m++] = t;
        if (t.src != t.dst) s[k++] = in_span(t.src, bytes);
        s[k++] = out_span(t.dst, bytes);
    };
    for (int i = 0; i < n_tensors; ++i) {
        const omega_grad_tensor &t = tensors[i];
        if (!dtype_ok(t.dtype) || t.reserved != 0 || t.n > ((uint64_t)1 << 48)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: bad dtype or length of a tensor");
        if (t.n == 0) continue;
        if (!t.src || !t.dst || misaligned(t.src, dtype_size(t.dtype)) || misaligned(t.dst, dtype_size(t.dtype)))
            OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: NULL or misaligned tensor");
        add(t);
    }
    for (int i = 0; i < n_layers; ++i) {
        if (!layers[i] || layers[i]->ctx != ctx) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: a layer is NULL or of another context");
        float *g;
        size_t len;
        if (!moe_grad_view(layers[i], &g, &len)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: no backward has run on a layer");
        add({g, g, len, OMEGA_DTYPE_F32, 0});
    }
    s[k++] = out_span(norm_out, norm_out ? 8 : 0);
    if (overlapping(s, k)) OMEGA_FAIL(ctx, OMEGA_ERR_INVALID_ARG, "clip_grad_norm: a tensor is there twice, or buffers overlap");
    void *ws;
    WORKSPACE(ctx, clip_workspace(all, m), &ws);
    OMEGA_HIP_CHECK(ctx, launch_clip(all, m, max_norm, norm_out, ws, ctx->stream));
    return OMEGA_OK;
}

}  // extern "C"
