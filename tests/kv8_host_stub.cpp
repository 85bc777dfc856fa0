// Stands in for the context and the HIP runtime under er_kv8.cpp, so that what
// the host does with a valid context runs without a device: launches are recorded.
#include "er_kv8_host.h"

#include <cstdarg>
#include <cstdio>

#include <vector>

extern "C" const unsigned char er_kv8_blob[1] = {0};

struct er_hip_ctx {
    er_detail::Kv8Kernels kernels;
    int cu;
};

namespace er_detail {
thread_local char g_last_error[512];
er_status fail(er_status st, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
    va_end(ap);
    return st;
}
const Kv8Kernels &kv8_of(const er_hip_ctx *ctx) { return ctx->kernels; }
int cu_count_of(const er_hip_ctx *ctx) { return ctx->cu; }
er_status bind_device_of(const er_hip_ctx *) { return ER_OK; }
}  // namespace er_detail

static bool g_loads = true;
static std::vector<unsigned> g_grids;

extern "C" {
hipError_t hipModuleLoadData(hipModule_t *m, const void *) {
    *m = g_loads ? (hipModule_t)1 : nullptr;
    return g_loads ? hipSuccess : hipErrorInvalidImage;
}
hipError_t hipModuleGetFunction(hipFunction_t *f, hipModule_t, const char *) { return *f = (hipFunction_t)1, hipSuccess; }
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "stub"; }
hipError_t hipModuleLaunchKernel(hipFunction_t, unsigned x, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned,
                                 hipStream_t, void **, void **) {
    g_grids.push_back(x);
    return hipSuccess;
}

er_hip_ctx *stub_create(int cu, int loads) {
    g_loads = loads != 0;
    er_hip_ctx *ctx = new er_hip_ctx{};
    ctx->cu = cu;
    (void)er_detail::kv8_load(ctx->kernels);
    return ctx;
}
void stub_destroy(er_hip_ctx *ctx) {
    er_detail::kv8_unload(ctx->kernels);
    delete ctx;
}
// The grids launched since the last call: how many, and the first two.
int stub_launches(unsigned *first, unsigned *second) {
    const int n = (int)g_grids.size();
    *first = n > 0 ? g_grids[0] : 0;
    *second = n > 1 ? g_grids[1] : 0;
    g_grids.clear();
    return n;
}
const char *stub_error() { return er_detail::g_last_error; }
}
