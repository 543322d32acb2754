// Checks of the arguments and the workspace of the operators on caller-owned buffers: shared by their C entries.
#pragma once
#include <algorithm>

#include "common.h"

static inline bool dtype_ok(int dt) { return dt == OMEGA_DTYPE_F32 || dt == OMEGA_DTYPE_BF16; }
static inline size_t dtype_size(int dt) { return dt == OMEGA_DTYPE_BF16 ? 2 : 4; }
#define SIZE_MAX_ROWS (1 << 30)  // sums of sizes stay within 32 bits; launches whose lanes would not are cut by the launchers
#define SIZE_MAX_COLS (1 << 20)
static inline bool sizes_ok(int T, int V, int d) { return T >= 0 && V >= 1 && d >= 1 && T <= SIZE_MAX_ROWS && V <= SIZE_MAX_ROWS && d <= SIZE_MAX_COLS; }

struct span {
    uintptr_t b, e;
    bool out;
    bool operator<(const span &o) const { return b < o.b; }
};
static inline span in_span(const void *p, size_t bytes) { return {(uintptr_t)p, (uintptr_t)p + bytes, false}; }
static inline span out_span(const void *p, size_t bytes) { return {(uintptr_t)p, (uintptr_t)p + bytes, true}; }

// Whether an output shares memory with anything else (sorts `s`)
static inline bool overlapping(span *s, int n)
{
    std::sort(s, s + n);
    uintptr_t end_in = 0, end_out = 0;
    for (int i = 0; i < n; ++i) {
        if (s[i].b == s[i].e) continue;
        if (s[i].b < end_out || (s[i].out && s[i].b < end_in)) return true;
        uintptr_t &end = s[i].out ? end_out : end_in;
        end = std::max(end, s[i].e);
    }
    return false;
}

static inline bool misaligned(const void *p, size_t to) { return (uintptr_t)p % to != 0; }

// The context's workspace, at least `bytes` of it
static inline int op_workspace(omega_ctx *ctx, size_t bytes, void **ws)
{
    if (bytes > ctx->op_ws_bytes) {
        OMEGA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
        if (ctx->op_ws) (void)hipFree(ctx->op_ws);
        ctx->op_ws = nullptr;
        ctx->op_ws_bytes = 0;
        const hipError_t e = hipMalloc(&ctx->op_ws, bytes);
        if (e != hipSuccess) {
            (void)hipGetLastError();  // the next launch would else report it as its own
            ctx->op_ws = nullptr;
            return omega_set_error(ctx, e == hipErrorOutOfMemory ? OMEGA_ERR_OOM : OMEGA_ERR_HIP, "workspace of the operator", e, __FILE__, __LINE__);
        }
        ctx->op_ws_bytes = bytes;
    }
    *ws = ctx->op_ws;
    return OMEGA_OK;
}

#define WORKSPACE(ctx, bytes, ws)                          \
    do {                                                   \
        const int _st = op_workspace((ctx), (bytes), (ws)); \
        if (_st != OMEGA_OK) return _st;                   \
    } while (0)
