// Stands in for the context and the HIP runtime under er_draft.cpp, so that what
// the host does with a valid context runs without a device: launches are
// recorded with their LDS.
#include "er_draft_host.h"

#include <cstdarg>
#include <cstdio>

#include <vector>

extern "C" const unsigned char er_draft_blob[1] = {0};

struct er_hip_ctx {
    er_detail::DraftKernels kernels;
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
const DraftKernels &draft_of(const er_hip_ctx *ctx) { return ctx->kernels; }
const Kv8Kernels &kv8_of(const er_hip_ctx *) {
    static const Kv8Kernels none;
    return none;
}
int cu_count_of(const er_hip_ctx *ctx) { return ctx->cu; }
er_status bind_device_of(const er_hip_ctx *) { return ER_OK; }
}  // namespace er_detail

static bool g_loads = true;
struct Launched {
    unsigned grid, lds;
};
static std::vector<Launched> g_launches;

extern "C" {
hipError_t hipModuleLoadData(hipModule_t *m, const void *) {
    *m = g_loads ? (hipModule_t)1 : nullptr;
    return g_loads ? hipSuccess : hipErrorInvalidImage;
}
hipError_t hipModuleGetFunction(hipFunction_t *f, hipModule_t, const char *) { return *f = (hipFunction_t)1, hipSuccess; }
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "stub"; }
hipError_t hipModuleLaunchKernel(hipFunction_t, unsigned x, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned lds,
                                 hipStream_t, void **, void **) {
    g_launches.push_back({x, lds});
    return hipSuccess;
}

er_hip_ctx *stub_create(int cu, int loads) {
    g_loads = loads != 0;
    er_hip_ctx *ctx = new er_hip_ctx{};
    ctx->cu = cu;
    (void)er_detail::draft_load(ctx->kernels);
    return ctx;
}
void stub_destroy(er_hip_ctx *ctx) {
    er_detail::draft_unload(ctx->kernels);
    delete ctx;
}
// The launches since the last call: how many; grid and LDS bytes of the first
// two.
int stub_launches(unsigned *out) {
    const int n = (int)g_launches.size();
    for (int i = 0; i < 2 && i < n; ++i) out[2 * i] = g_launches[i].grid, out[2 * i + 1] = g_launches[i].lds;
    g_launches.clear();
    return n;
}
const char *stub_error() { return er_detail::g_last_error; }
}
