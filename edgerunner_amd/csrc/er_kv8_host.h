// er_kv8_host.h -- the 8-bit cache's kernels of one context, shared by the
// host translation units (er_hip.cpp owns the context, er_kv8.cpp launches).
#pragma once

#include "er_error.h"

#include <hip/hip_runtime_api.h>

namespace er_detail {

constexpr int kKv8Dims = 3;   // head widths 64, 128, 256
constexpr int kKv8Pages = 3;  // pages of 16, 32, 64 tokens

struct Kv8Kernels {
    hipModule_t module = nullptr;
    hipFunction_t rope[kKv8Dims] = {}, append[kKv8Dims] = {}, join[kKv8Dims] = {}, joinRow[kKv8Dims] = {};
    hipFunction_t narrow[kKv8Dims][kKv8Pages][2] = {}, wide[kKv8Dims][kKv8Pages][2] = {};  // [fp32, bf16 output]
};

// Loads the cache's code object on the current device and resolves its kernels;
// where it fails, nothing of it stays.
er_status kv8_load(Kv8Kernels &k);
void kv8_unload(Kv8Kernels &k);

// Of a context that is not null: its kernels, its compute units, and the
// device made current.
const Kv8Kernels &kv8_of(const er_hip_ctx *ctx);
int cu_count_of(const er_hip_ctx *ctx);
er_status bind_device_of(const er_hip_ctx *ctx);

}  // namespace er_detail
