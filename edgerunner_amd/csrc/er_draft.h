// er_draft.h -- kernel arguments of what a step does with drafted tokens and
// with logits (er_draft.hip), shared with the host (er_draft.cpp).
#pragma once

#include "er_kv8.h"

#define ER_FEW_LEAST 4u  // 64-token steps that a share of an attention call has at least; half where they fit half the workgroups
#define ER_CHOOSE_THREADS 256
#define ER_CHOOSE_SLICE (8 * ER_CHOOSE_THREADS)  // tokens of a workgroup; half below a vocabulary of as many

struct ErAcceptArgs {
    ErKv8Cache c;
    ErKv8Batch b;
    const int32_t *parent, *token, *chosen;  // [rows]
    int32_t *path;                           // [rows]
    int32_t *count, *next, *left;            // [sequences]
};

struct ErChooseArgs {
    const float *logits;
    float *out;               // null: not written
    int32_t *chosen;          // null: not found
    float *partV;             // [rows][slices]: the largest allowed of a slice
    uint32_t *partI;          // and its token
    const int32_t *start;     // null: row r is sequence r
    const int32_t *history, *historyLen;
    const float *penalty;     // [sequences][3]
    const int32_t *biasToken, *biasLen;
    const float *bias;
    const uint32_t *allowed;  // null: all
    const uint32_t *seen;     // null: no drafts
    const int32_t *token;
    uint32_t rows, maxRows, sequences, vocab, stride;
    uint32_t historyStride, biasStride, allowedStride, words;
    uint32_t slices;          // workgroups of a row
};
