// er_draft_host.h -- the kernels of er_draft.hip of one context, shared by the
// host translation units (er_hip.cpp owns the context, er_draft.cpp launches).
#pragma once

#include "er_kv8_host.h"

namespace er_detail {

struct DraftKernels {
    hipModule_t module = nullptr;
    hipFunction_t narrow[kKv8Dims][kKv8Pages][2] = {}, wide[kKv8Dims][kKv8Pages][2] = {};  // [fp32, bf16 output]
    hipFunction_t join[kKv8Dims] = {}, joinRow[kKv8Dims] = {}, accept[kKv8Dims] = {};
    hipFunction_t choose = nullptr, chooseJoin = nullptr;
};

// Loads the code object on the current device and resolves its kernels; where
// it fails, nothing of it stays.
er_status draft_load(DraftKernels &k);
void draft_unload(DraftKernels &k);

// Of a context that is not null.
const DraftKernels &draft_of(const er_hip_ctx *ctx);

}  // namespace er_detail
