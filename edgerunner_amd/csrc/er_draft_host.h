// er_draft_host.h -- the kernels of er_draft.hip of one context, shared by the
// host translation units (er_hip.cpp owns the context, er_draft.cpp launches).
#pragma once

#include "er_kv8_host.h"

namespace er_detail {

struct DraftKernels {
    hipModule_t module = nullptr;
    // [16, 32 columns a wave][..][..][fp32, bf16 output]; 32 up to width 128
    hipFunction_t few[2][kKv8Dims][kKv8Pages][2] = {}, wide[kKv8Dims][kKv8Pages][2] = {};
    hipFunction_t joinFew[2][kKv8Dims] = {}, joinColumn[2][kKv8Dims] = {}, join[kKv8Dims] = {}, joinRow[kKv8Dims] = {};
    hipFunction_t accept[kKv8Dims] = {};
    hipFunction_t choose[2] = {}, chooseJoin = nullptr;  // half slices, slices
};

// Loads the code object on the current device and resolves its kernels; where
// it fails, nothing of it stays.
er_status draft_load(DraftKernels &k);
void draft_unload(DraftKernels &k);

// Of a context that is not null.
const DraftKernels &draft_of(const er_hip_ctx *ctx);

}  // namespace er_detail
