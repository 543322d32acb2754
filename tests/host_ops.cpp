// Stand-ins for the launchers of the operators around the layer (ops_api.hip), beside those of host_runtime.cpp: what would be
// launched is a line of a log of its own, with the workspace that the launch was given.
#include <stdio.h>

#include <string>

#include "common.h"

static std::string g_ops;
static hipError_t op(const char *name, const void *ws, size_t bytes)
{
    char buf[96];
    snprintf(buf, sizeof buf, "%s ws=%d bytes=%zu\n", name, ws != nullptr, bytes);
    g_ops += buf;
    return hipSuccess;
}
extern "C" const char *host_take_ops(void)
{
    static std::string taken;
    taken.swap(g_ops);
    g_ops.clear();
    return taken.c_str();
}
extern "C" hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int) { return hipSuccess; }

hipError_t launch_embedding_forward(const void *, int, int, int, const int32_t *, int, float, void *, hipStream_t) { return op("lookup", nullptr, 0); }
size_t embedding_backward_workspace(int V, int d, int T) { return (size_t)V * 4 + (size_t)T * 8 + (size_t)d; }
hipError_t launch_embedding_backward(const int32_t *, int, const void *, int, int, int, float, bool, void *, int, void *ws, hipStream_t) { return op("gradient", ws, 0); }
hipError_t launch_layernorm_forward(const omega_ctx *, const void *, int, int, int, const float *, const float *, float, void *, float *, float *, hipStream_t) { return op("norm", nullptr, 0); }
size_t layernorm_backward_workspace(const omega_ctx *, int, int d) { return (size_t)d * 8; }
hipError_t launch_layernorm_backward(const omega_ctx *, const void *, const void *, int, int, int, const float *, const float *, const float *, void *, float *, float *, void *ws,
                                     hipStream_t)
{
    return op("norm_back", ws, 0);
}
size_t head_workspace(const omega_ctx *, const head_args &a, bool backward) { return (size_t)a.T * (backward ? 4096 : 1024); }
hipError_t launch_head_forward(const omega_ctx *, const head_args &, void *ws, hipStream_t) { return op("head", ws, 0); }
hipError_t launch_head_backward(const omega_ctx *, const head_args &, void *ws, hipStream_t) { return op("head_back", ws, 0); }
hipError_t head_init(void) { return hipSuccess; }
size_t clip_workspace(const omega_grad_tensor *t, int n)
{
    size_t b = 256;
    for (int i = 0; i < n; ++i) b += t[i].n;
    return b;
}
hipError_t launch_clip(const omega_grad_tensor *t, int n, float, float *, void *ws, hipStream_t) { return op("clip", ws, clip_workspace(t, n)); }
