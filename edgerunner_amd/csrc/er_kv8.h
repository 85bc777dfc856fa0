// er_kv8.h -- kernel arguments of the 8-bit cache's operators, shared by the
// kernels (er_kv8.hip) and the host (er_kv8.cpp).  Plain values and device
// pointers, passed by value.
#pragma once

#include <stdint.h>

#define ER_KV8_THREADS 256
#define ER_MOST_DRAFTS 1024  // rows of a sequence that are drafts
#define ER_KV8_ROW_PARTS 16  // parts that the join of a whole row takes at the most

// Norm and rotation of one kind of heads.
struct ErTurn {
    const float *in;
    float *out;
    const float *norm;   // null: none
    uint32_t inStride;
    uint32_t outStride;
    uint32_t heads;
};

struct ErRopeArgs {
    ErTurn q, k;              // k.heads == 0: queries alone
    const int32_t *positions;
    const float *freq;
    uint32_t rot, pairs;      // rotated width; neighbours rather than halves
    uint32_t rows;
    uint32_t chunks;          // waves a row is cut into
    float eps;
};

struct ErKv8Cache {
    uint8_t *k, *v;
    float *ks, *vs;
    uint32_t pages, heads, shift;  // shift: log2 of the tokens a page holds
};

struct ErKv8Batch {
    const int32_t *table, *len, *start;
    uint32_t sequences, stride, rows, maxRows;
    uint32_t maxLen;  // min(max_kv_len, stride * page tokens)
};

struct ErAppendArgs {
    ErKv8Cache c;
    ErKv8Batch b;
    const float *k;
    const void *v;
    const float *kNorm;
    uint32_t kStride, vStride, vHalf;
    ErTurn q;                 // q.heads == 0: none ride along
    const float *freq;
    uint32_t rot, pairs;
    uint32_t spans;           // pages that max_rows rows of a sequence can touch
    uint32_t cacheBlocks;     // workgroups that write the cache; the ones behind take the queries
    uint32_t chunks;          // of the queries, as in ErRopeArgs
    float eps;
};

struct ErAttendArgs {
    static constexpr bool MASKED = false;
    ErKv8Cache c;
    ErKv8Batch b;
    const float *q;
    void *out;
    float *partO;             // fp32 [parts][head_dim]: sums of columns whose tokens several workgroups share
    float *partML;            // fp32 [parts][2]: their reference exponents and sums of weights
    uint32_t qStride, outStride;
    uint32_t group;           // query heads of one key/value head
    // narrow kernel: workgroups that share the tokens of all sequences evenly,
    // at least `least` 64-token steps each (0: a workgroup a
    // sequence, head and block of 16 columns)
    uint32_t shares, least;
    // wide kernel: pieces of a row tile's tokens, tokens of a piece (a multiple
    // of 64), row tiles of a sequence and key/value head (narrow kernel: blocks
    // of 16 columns)
    uint32_t splits, chunk, tiles;
    uint32_t window;          // 0: none
    uint32_t half;            // bf16 output
    float scale;              // times log2(e)
};

// Attention where not every earlier token is visible.
struct ErMaskedArgs : ErAttendArgs {
    static constexpr bool MASKED = true;
    const uint32_t *seen;     // [rows][words]: bit j, the sequence's row j is visible; null: no drafts, the rows are causal
    const int32_t *position;  // [rows]; read where there are drafts and a window
    uint32_t words;
    uint32_t sinks;           // first tokens that stay visible
};
