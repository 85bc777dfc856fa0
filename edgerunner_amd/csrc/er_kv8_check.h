// er_kv8_check.h -- what the host sides of the operators over the 8-bit cache
// (er_kv8.cpp, er_draft.cpp) share: checks of arguments, kernel arguments,
// how an attention call is cut up, launches.
#pragma once

#include "er_hip.h"
#include "er_kv8.h"
#include "er_kv8_host.h"

#include <algorithm>

namespace er_detail {

constexpr uint32_t kMostHeads = 65536;  // heads and strides that keep 32-bit indices inside a row

typedef unsigned long long ull;

inline bool misaligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

inline int dim_index(uint32_t d) { return d == 64 ? 0 : d == 128 ? 1 : d == 256 ? 2 : -1; }

inline er_status check_dim(const char *op, uint32_t d) {
    if (dim_index(d) < 0) return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: head_dim %u is not 64, 128 or 256", op, d);
    return ER_OK;
}

inline er_status check_buffer(const char *op, const char *what, const er_buffer &b, uint64_t need, uintptr_t align,
                       er_status shortage = ER_ERR_ENCODING_FAILED) {
    if (b.length < need)
        return fail(shortage, "%s: %s too small: %llu B (needs %llu)", op, what, (ull)b.length, (ull)need);
    if (!b.data) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null %s", op, what);
    if (misaligned(b.data, align))
        return fail(ER_ERR_INVALID_ARGUMENT, "%s: %s must be %u-byte aligned", op, what, (unsigned)align);
    return ER_OK;
}

inline er_status check_rows(const char *op, const char *what, const er_head_rows *h, uint32_t rows, uint32_t d,
                     uint32_t bytes) {
    if (!h) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null %s", op, what);
    if (h->heads == 0 || h->heads > kMostHeads)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %s has %u heads (1 .. %u)", op, what, h->heads, kMostHeads);
    if ((uint64_t)h->heads * d > h->row_stride)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %s row stride %u holds no %u heads of %u", op, what,
                    h->row_stride, h->heads, d);
    return check_buffer(op, what, h->data, ((uint64_t)(rows - 1) * h->row_stride + (uint64_t)h->heads * d) * bytes,
                        bytes);
}

// Two row buffers that the kernel may read and write at once: the same heads
// at the same places, or apart.
inline er_status check_apart(const char *op, const char *what, const er_head_rows *in, const er_head_rows *out,
                      uint32_t rows, uint32_t d, uint32_t inBytes, uint32_t outBytes, bool mayBeSame) {
    if (mayBeSame && in->data.data == out->data.data && in->row_stride == out->row_stride && in->heads == out->heads)
        return ER_OK;
    const uintptr_t a = (uintptr_t)in->data.data, b = (uintptr_t)out->data.data;
    const uint64_t na = ((uint64_t)(rows - 1) * in->row_stride + (uint64_t)in->heads * d) * inBytes;
    const uint64_t nb = ((uint64_t)(rows - 1) * out->row_stride + (uint64_t)out->heads * d) * outBytes;
    if (a + na <= b || b + nb <= a) return ER_OK;
    // columns of one wider row: equal strides, and the two windows of a row apart, around the row's end too
    if (in->row_stride == out->row_stride && inBytes == outBytes) {
        const uint64_t row = (uint64_t)in->row_stride * inBytes, wa = (uint64_t)in->heads * d * inBytes,
                       wb = (uint64_t)out->heads * d * outBytes;
        const uint64_t ahead = a <= b ? (b - a) % row : (row - (a - b) % row) % row;  // b's window behind a's
        if (ahead >= wa && ahead + wb <= row) return ER_OK;
    }
    return fail(ER_ERR_INVALID_ARGUMENT, "%s: %s overlap", op, what);
}

inline er_status check_cache(const char *op, const er_kv8_cache *c) {
    if (!c) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null cache", op);
    er_status st = check_dim(op, c->head_dim);
    if (st != ER_OK) return st;
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: page_tokens %u is not 16, 32 or 64", op, c->page_tokens);
    if (c->kv_heads == 0 || c->kv_heads > kMostHeads)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u key/value heads (1 .. %u)", op, c->kv_heads, kMostHeads);
    if (c->pages == 0 || c->pages > 0x7fffffffu)
        return fail(ER_ERR_INVALID_MATRIX_SHAPE, "%s: %u pages", op, c->pages);
    const uint64_t blocks = (uint64_t)c->pages * c->kv_heads, codes = (uint64_t)c->page_tokens * c->head_dim;
    // blocks < 2^47 and codes <= 2^14, so the products stay inside 64 bits
    st = check_buffer(op, "k cache", c->k, blocks * codes, 16, ER_ERR_INVALID_MATRIX_SHAPE);
    if (st == ER_OK) st = check_buffer(op, "v cache", c->v, blocks * codes, 16, ER_ERR_INVALID_MATRIX_SHAPE);
    if (st == ER_OK) st = check_buffer(op, "k scales", c->k_scale, blocks * 4, 4, ER_ERR_INVALID_MATRIX_SHAPE);
    if (st == ER_OK) st = check_buffer(op, "v scales", c->v_scale, blocks * 4, 4, ER_ERR_INVALID_MATRIX_SHAPE);
    return st;
}

inline er_status check_batch(const char *op, const er_kv8_batch *b) {
    if (!b) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null batch", op);
    // indices of rows and tokens are signed 32-bit in the kernels
    if (b->rows > 0x3fffffffu || b->sequences > 0x3fffffffu || b->max_kv_len > 0x3fffffffu || b->table_stride > 0x3fffffffu)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: batch of %u sequences, %u rows, %u tokens, table of %u: over 2^30",
                    op, b->sequences, b->rows, b->max_kv_len, b->table_stride);
    if (b->rows == 0 || b->sequences == 0) return ER_OK;  // nothing to do, nothing read
    if (b->max_rows == 0 || b->max_rows > b->rows)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: max_rows %u of %u rows", op, b->max_rows, b->rows);
    er_status st = check_buffer(op, "page table", b->page_table, (uint64_t)b->sequences * b->table_stride * 4, 4);
    if (st == ER_OK) st = check_buffer(op, "kv_len", b->kv_len, (uint64_t)b->sequences * 4, 4);
    if (st == ER_OK) st = check_buffer(op, "row_start", b->row_start, ((uint64_t)b->sequences + 1) * 4, 4);
    return st;
}

inline uint32_t most_tokens(const er_kv8_cache *c, const er_kv8_batch *b) {
    return (uint32_t)std::min<uint64_t>(b->max_kv_len, (uint64_t)b->table_stride * c->page_tokens);
}

inline ErKv8Cache cache_args(const er_kv8_cache *c) {
    ErKv8Cache a{};
    a.k = (uint8_t *)c->k.data, a.v = (uint8_t *)c->v.data;
    a.ks = (float *)c->k_scale.data, a.vs = (float *)c->v_scale.data;
    a.pages = c->pages, a.heads = c->kv_heads;
    a.shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : 6;
    return a;
}

inline ErKv8Batch batch_args(const er_kv8_cache *c, const er_kv8_batch *b) {
    ErKv8Batch a{};
    a.table = (const int32_t *)b->page_table.data;
    a.len = (const int32_t *)b->kv_len.data;
    a.start = (const int32_t *)b->row_start.data;
    a.sequences = b->sequences, a.stride = b->table_stride, a.rows = b->rows, a.maxRows = b->max_rows;
    a.maxLen = most_tokens(c, b);
    return a;
}

// Kernels count a launch's threads in 32 bits.
constexpr uint64_t kMostBlocks = (1ull << 32) / ER_KV8_THREADS - 1;

inline er_status check_blocks(const char *op, uint64_t blocks) {
    if (blocks > kMostBlocks)
        return fail(ER_ERR_ENCODING_FAILED, "%s: %llu workgroups exceed a launch", op, (ull)blocks);
    return ER_OK;
}

inline er_status launch(hipFunction_t f, const char *op, uint64_t blocks, uint32_t lds, er_stream stream, void *args) {
    const er_status st = check_blocks(op, blocks);
    if (st != ER_OK) return st;
    void *params[] = {args};
    const hipError_t e = hipModuleLaunchKernel(f, (uint32_t)blocks, 1, 1, ER_KV8_THREADS, 1, 1, lds,
                                               (hipStream_t)stream, params, nullptr);
    if (e != hipSuccess) return fail(ER_ERR_ENCODING_FAILED, "hipModuleLaunchKernel(%s): %s", op, hipGetErrorString(e));
    return ER_OK;
}

inline er_status check_ctx(const er_hip_ctx *ctx) {
    return ctx ? ER_OK : fail(ER_ERR_INVALID_ARGUMENT, "null er_hip_ctx");
}

// How an attention call is cut up.
struct AttendPlan {
    bool narrow;
    uint32_t shares, least;         // narrow kernel
    uint32_t tiles, splits, chunk;  // wide kernel
    uint64_t parts;                 // columns that the workspace holds sums of, at the most over all windows
};

// Columns (rows times query heads of a key/value head) decide the kernel.  The
// narrow one reads the cache once for each 16 of them, the wide one once for
// 128, with products that pay for columns that are not there, and with less
// work split between fewer workgroups.  Measured narrow / wide, us: 24 columns
// of 4 sequences of 30000 tokens 27 / 37, 32 of 16 of 8000 in bf16 59 / 85, 60
// of 16 of 4000 25 / 56, but 128 of 4 of 8000 51 / 43 and of 16 of 4000 98 / 73.
// At head width 256 the wide one has a wave a SIMD: 32 of 16 of 8000 63 / 166,
// 100 of 8 of 4000 50 / 63.
inline AttendPlan plan_attend(const er_kv8_cache *c, const er_kv8_batch *b, uint32_t group, uint32_t window, int cu,
                              uint32_t sinks = 0, bool drafts = false) {
    AttendPlan p{};
    const uint64_t cols = (uint64_t)b->max_rows * group, full = most_tokens(c, b);
    p.narrow = cols <= (c->head_dim == 256 ? 128 : 64);
    p.splits = 1;
    if (p.narrow) {
        // two workgroups a CU are resident; a workgroup's start and its part in the join cost as much as some
        // hundred tokens, so none takes fewer than that, and what a workgroup
        // a sequence and head reads in that time is not shared at all.  By 1, 2, 4 and 8 steps of 64 tokens, us: 16
        // draft checks at head width 256 (17 steps a unit) 26.2, 26.2, 20.7, 21.3; a user of 8000 tokens at width 128
        // 19.4, 17.0, 13.9, 14.6; 16 of up to 4000 at width 64 15.2, 15.5, 13.6, 13.5
        const uint64_t resident = (uint64_t)cu * 2;
        p.tiles = (uint32_t)((cols + 15) / 16);
        if (full > 512) {
            p.shares = (uint32_t)resident;
            p.least = 4;
            p.parts = 2 * resident * 16;
        }
        return p;
    }
    p.tiles = (uint32_t)((cols + 127) / 128);
    uint64_t span = full;
    // the tile's rows see window + rows - 1 tokens, and pieces begin at a multiple of 64; windows of drafts begin anywhere
    // among all rows' own; sinks take whole steps of their own
    if (window)
        span = std::min<uint64_t>(span, (uint64_t)window + (drafts ? b->max_rows : 128 / group + 2) + 63 + (((uint64_t)sinks + 63) & ~63ull));
    // The tokens of a (sequence, head, row tile) are cut into as many pieces as
    // make one workgroup for each that the chip holds, of 256 tokens at the
    // least: fewer leave it empty, more have more sums to join (bf16, a chunk of 256
    // rows behind 60000 tokens in 4, 8, 12 and 16 pieces a tile 384, 323, 339 and 337
    // us; a prompt of 4096 rows of 8 heads in one and two 193 and 284).  Of a
    // prompt's pieces half lie behind its rows, and of several sequences one
    // eighth behind their ends: a guess, since lengths are known on the device
    // alone.  Three ragged chunks take 86 us in 5 pieces, 73 in 7, 78 in 8 and in 10; the rule takes 8.
    const uint64_t resident = (uint64_t)cu * (c->head_dim == 64 ? 3 : c->head_dim == 128 ? 2 : 1);
    const uint64_t filled = std::max<uint64_t>(1, ((uint64_t)b->rows * group + 64ull * b->sequences) / 128);
    const uint64_t units = c->kv_heads * std::min(filled, (uint64_t)b->sequences * p.tiles);
    auto pieces = [&](uint64_t tokens, bool windowed) {
        const double rows = (double)std::min<uint64_t>(b->max_rows, full), length = (double)std::max<uint64_t>(1, full);
        double seen = windowed ? 1.0 : 1.0 - 0.5 * rows / length;
        if (b->sequences > 1) seen *= 0.875;
        const uint64_t even = (uint64_t)((double)resident / ((double)units * seen) + 0.5);
        return std::max<uint64_t>(1, std::min<uint64_t>(even, (tokens + 255) / 256));
    };
    const uint64_t splits = pieces(span, span < full);
    p.chunk = (uint32_t)std::max<uint64_t>(64, ((span + splits - 1) / splits + 63) & ~63ull);
    p.splits = (uint32_t)std::max<uint64_t>(1, (span + p.chunk - 1) / p.chunk);
    // no window has more pieces than the whole length, and rounding them up to 64 tokens only takes some away
    const uint64_t most = pieces(full, false);
    if (most > 1) p.parts = most * b->rows * group * c->kv_heads;
    return p;
}

inline er_status check_group(const char *op, const er_kv8_cache *c, const er_kv8_batch *b, uint32_t qHeads) {
    if (qHeads == 0 || qHeads % c->kv_heads != 0 || qHeads / c->kv_heads > 1024)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u query heads over %u key/value heads", op, qHeads, c->kv_heads);
    // columns of a sequence, and 64-token steps of all sequences and heads (rounded up to four each, for up to eight column
    // blocks), are 32-bit counts
    const uint64_t steps = (uint64_t)b->sequences * ((most_tokens(c, b) + 63u) / 64u + 4u);
    if ((uint64_t)b->max_rows * (qHeads / c->kv_heads) > 0x7fffffffull || steps > 0x0fffffffull / c->kv_heads)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u sequences of up to %u tokens and %u rows: too many to count in 31 bits",
                    op, b->sequences, most_tokens(c, b), b->max_rows);
    return ER_OK;
}

// How the parts of an attention call are joined.
struct JoinLaunch {
    hipFunction_t f;
    uint64_t blocks;
    uint32_t lds;
};
// After the wide kernel, a workgroup a row where the parts are few; else one a
// row and head.
inline JoinLaunch join_of(const AttendPlan &p, hipFunction_t join, hipFunction_t joinRow, uint32_t rows, uint32_t heads) {
    if (!p.shares && p.splits <= ER_KV8_ROW_PARTS) return JoinLaunch{joinRow, rows, 0};
    return JoinLaunch{join, (uint64_t)rows * heads, (4 * ER_KV8_THREADS + (p.shares ? p.shares : p.splits)) * 4};
}

// The launches of an attention call whose other arguments are in `a`.
template <class ARGS>
er_status launch_attend(const char *op, hipFunction_t attend, const JoinLaunch &join, ARGS &a, const AttendPlan &p, uint32_t d,
                        const er_buffer &workspace, er_stream stream) {
    const bool joined = p.splits > 1 || p.shares > 0;
    er_status st = ER_OK;
    if (joined) {
        st = check_buffer(op, "workspace", workspace, p.parts * (d + 2) * 4, 16);
        if (st != ER_OK) return st;
        a.partO = (float *)workspace.data;
        a.partML = a.partO + p.parts * d;
    }
    const uint64_t pairs = (uint64_t)a.b.sequences * a.c.heads;
    const uint64_t blocks = p.shares ? p.shares : pairs * p.splits * p.tiles;  // narrow: one split
    // both, before the first is queued
    st = check_blocks(op, blocks);
    if (st == ER_OK && joined) st = check_blocks(op, join.blocks);
    if (st != ER_OK) return st;
    st = launch(attend, op, blocks, 0, stream, &a);
    if (st != ER_OK || !joined) return st;
    return launch(join.f, op, join.blocks, join.lds, stream, &a);
}

}  // namespace er_detail
