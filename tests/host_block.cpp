// Stand-ins for the launchers of the operators around the experts (block_api.hip), beside those of host_runtime.cpp and host_ops.cpp; what
// would be launched is a line of a log of its own.
#include <stdio.h>

#include <string>

#include "common.h"

static std::string g_block;
static hipError_t op(const char *name, const void *ws = nullptr)
{
    g_block += name;
    g_block += ws ? " ws\n" : "\n";
    return hipSuccess;
}
extern "C" const char *host_take_block(void)
{
    static std::string taken;
    taken.swap(g_block);
    g_block.clear();
    return taken.c_str();
}
hipError_t launch_rmsnorm_forward(const omega_ctx *, const rmsnorm_forward &, hipStream_t) { return op("rms"); }
size_t rmsnorm_backward_workspace(const omega_ctx *, int, int d) { return (size_t)d * 4; }
hipError_t launch_rmsnorm_backward(const omega_ctx *, const rmsnorm_backward &, void *ws, hipStream_t) { return op("rms_back", ws); }
hipError_t launch_keep8_save(const void *, int, int, int, int, uint8_t *, void *, hipStream_t) { return op("save"); }
hipError_t launch_keep8_load(const uint8_t *, const void *, int, int, int, void *, int, hipStream_t) { return op("load"); }
size_t route_workspace(const omega_ctx *, const omega_route_config &c, int T) { return (size_t)(T + 1) * c.E * 4; }
hipError_t launch_route_forward(const omega_ctx *, const omega_route_config &, const float *, int, const float *, int32_t *, float *, int32_t *, void *ws, hipStream_t) { return op("route", ws); }
hipError_t launch_route_backward(const omega_route_config &, const float *, int, const int32_t *, const float *, const float *, float *, hipStream_t) { return op("route_back"); }
hipError_t launch_route_balance(const int32_t *, int, float, float *, hipStream_t) { return op("balance"); }
