// er_kv8.cpp -- host side of the operators between the projections (head norms
// with the rotation, the 8-bit paged cache, attention over it): checks of
// arguments, launch plans, launches.  Nothing here allocates or synchronises,
// so every call can be recorded into a graph.
#include "er_hip.h"
#include "er_kv8.h"
#include "er_kv8_host.h"

#include <algorithm>
#include <cmath>
#include <cstdio>

extern "C" const unsigned char er_kv8_blob[];

namespace er_detail {

er_status kv8_load(Kv8Kernels &k) {
    hipError_t e = hipModuleLoadData(&k.module, er_kv8_blob);
    if (e != hipSuccess) {
        k.module = nullptr;
        return fail(ER_ERR_LIBRARY_NOT_FOUND, "hipModuleLoadData(cache kernels): %s", hipGetErrorString(e));
    }
    static const int dims[kKv8Dims] = {64, 128, 256};
    static const char *const outs[2] = {"f32", "bf16"};
    auto find = [&](hipFunction_t &f, const char *name) {
        const hipError_t r = hipModuleGetFunction(&f, k.module, name);
        if (r == hipSuccess) return ER_OK;
        return fail(ER_ERR_FUNCTION_NOT_FOUND, "functionNotFound(%s): %s", name, hipGetErrorString(r));
    };
    er_status st = ER_OK;
    for (int d = 0; d < kKv8Dims && st == ER_OK; ++d) {
        char name[64];
        auto named = [&](const char *form, int page, const char *out) {
            std::snprintf(name, sizeof(name), form, dims[d], page, out);
            return name;
        };
        st = find(k.rope[d], named("er_qk_norm_rope_d%d", 0, ""));
        if (st == ER_OK) st = find(k.append[d], named("er_kv8_append_d%d", 0, ""));
        if (st == ER_OK) st = find(k.join[d], named("er_kv8_join_d%d", 0, ""));
        if (st == ER_OK) st = find(k.joinRow[d], named("er_kv8_join_row_d%d", 0, ""));
        for (int i = 0; i < kKv8Pages * 2 && st == ER_OK; ++i) {
            const int page = i / 2, out = i % 2;
            st = find(k.narrow[d][page][out], named("er_kv8_attend_narrow_d%d_p%d_%s", 16 << page, outs[out]));
            if (st == ER_OK) st = find(k.wide[d][page][out], named("er_kv8_attend_wide_d%d_p%d_%s", 16 << page, outs[out]));
        }
    }
    if (st != ER_OK) kv8_unload(k);
    return st;
}

void kv8_unload(Kv8Kernels &k) {
    if (k.module) (void)hipModuleUnload(k.module);
    k = Kv8Kernels{};
}

}  // namespace er_detail

namespace {

using namespace er_detail;

constexpr uint32_t kMostHeads = 65536;  // heads and strides that keep 32-bit indices inside a row

typedef unsigned long long ull;

bool misaligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

int dim_index(uint32_t d) { return d == 64 ? 0 : d == 128 ? 1 : d == 256 ? 2 : -1; }

er_status check_dim(const char *op, uint32_t d) {
    if (dim_index(d) < 0) return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: head_dim %u is not 64, 128 or 256", op, d);
    return ER_OK;
}

er_status check_buffer(const char *op, const char *what, const er_buffer &b, uint64_t need, uintptr_t align,
                       er_status shortage = ER_ERR_ENCODING_FAILED) {
    if (b.length < need)
        return fail(shortage, "%s: %s too small: %llu B (needs %llu)", op, what, (ull)b.length, (ull)need);
    if (!b.data) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null %s", op, what);
    if (misaligned(b.data, align))
        return fail(ER_ERR_INVALID_ARGUMENT, "%s: %s must be %u-byte aligned", op, what, (unsigned)align);
    return ER_OK;
}

er_status check_rows(const char *op, const char *what, const er_head_rows *h, uint32_t rows, uint32_t d,
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
er_status check_apart(const char *op, const char *what, const er_head_rows *in, const er_head_rows *out,
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

er_status check_rope(const char *op, const er_rope *r, uint32_t d) {
    if (!r) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null rope", op);
    if (r->rotary_dim % 8 != 0 || r->rotary_dim > d)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: rotary_dim %u is no multiple of 8 up to %u", op, r->rotary_dim, d);
    if (r->rotary_dim == 0) return ER_OK;
    return check_buffer(op, "inv_freq", r->inv_freq, (uint64_t)(r->rotary_dim / 2) * 4, 4);
}

er_status check_norm(const char *op, const char *what, const er_buffer &w, uint32_t d) {
    return w.data ? check_buffer(op, what, w, (uint64_t)d * 4, 4) : ER_OK;
}

er_status check_cache(const char *op, const er_kv8_cache *c) {
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

er_status check_batch(const char *op, const er_kv8_batch *b) {
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

uint32_t most_tokens(const er_kv8_cache *c, const er_kv8_batch *b) {
    return (uint32_t)std::min<uint64_t>(b->max_kv_len, (uint64_t)b->table_stride * c->page_tokens);
}

ErKv8Cache cache_args(const er_kv8_cache *c) {
    ErKv8Cache a{};
    a.k = (uint8_t *)c->k.data, a.v = (uint8_t *)c->v.data;
    a.ks = (float *)c->k_scale.data, a.vs = (float *)c->v_scale.data;
    a.pages = c->pages, a.heads = c->kv_heads;
    a.shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : 6;
    return a;
}

ErKv8Batch batch_args(const er_kv8_cache *c, const er_kv8_batch *b) {
    ErKv8Batch a{};
    a.table = (const int32_t *)b->page_table.data;
    a.len = (const int32_t *)b->kv_len.data;
    a.start = (const int32_t *)b->row_start.data;
    a.sequences = b->sequences, a.stride = b->table_stride, a.rows = b->rows, a.maxRows = b->max_rows;
    a.maxLen = most_tokens(c, b);
    return a;
}

ErTurn turn_args(const er_head_rows *in, const er_head_rows *out, const er_buffer &norm) {
    ErTurn t{};
    t.in = (const float *)in->data.data, t.out = (float *)out->data.data;
    t.norm = (const float *)norm.data;
    t.inStride = in->row_stride, t.outStride = out->row_stride, t.heads = in->heads;
    return t;
}

// Kernels count a launch's threads in 32 bits.
constexpr uint64_t kMostBlocks = (1ull << 32) / ER_KV8_THREADS - 1;

er_status check_blocks(const char *op, uint64_t blocks) {
    if (blocks > kMostBlocks)
        return fail(ER_ERR_ENCODING_FAILED, "%s: %llu workgroups exceed a launch", op, (ull)blocks);
    return ER_OK;
}

er_status launch(hipFunction_t f, const char *op, uint64_t blocks, uint32_t lds, er_stream stream, void *args) {
    const er_status st = check_blocks(op, blocks);
    if (st != ER_OK) return st;
    void *params[] = {args};
    const hipError_t e = hipModuleLaunchKernel(f, (uint32_t)blocks, 1, 1, ER_KV8_THREADS, 1, 1, lds,
                                               (hipStream_t)stream, params, nullptr);
    if (e != hipSuccess) return fail(ER_ERR_ENCODING_FAILED, "hipModuleLaunchKernel(%s): %s", op, hipGetErrorString(e));
    return ER_OK;
}

er_status check_ctx(const er_hip_ctx *ctx) {
    return ctx ? ER_OK : fail(ER_ERR_INVALID_ARGUMENT, "null er_hip_ctx");
}

// The context's device current, its kernels there.
er_status make_ready(const char *op, const er_hip_ctx *ctx) {
    const er_status st = check_ctx(ctx);
    if (st != ER_OK) return st;
    if (!kv8_of(ctx).module) return fail(ER_ERR_LIBRARY_NOT_FOUND, "%s: the cache kernels did not load with this context", op);
    return bind_device_of(ctx);
}

// Waves that a row's strips of heads are cut into: with few rows one strip a
// wave (the shortest chain), with many as few as keep 16 waves a CU, so that a
// row's angles are formed as seldom as they can be.
uint32_t row_chunks(uint32_t strips, uint32_t rows, int cu) {
    const uint64_t want = (uint64_t)cu * 16;
    return (uint32_t)std::min<uint64_t>(strips, std::max<uint64_t>(1, want / rows));
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
AttendPlan plan_attend(const er_kv8_cache *c, const er_kv8_batch *b, uint32_t group, uint32_t window, int cu) {
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
    // the tile's rows see window + rows - 1 tokens, and pieces begin at a multiple of 64
    if (window) span = std::min<uint64_t>(span, (uint64_t)window + 128 / group + 2 + 63);
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

er_status check_group(const char *op, const er_kv8_cache *c, const er_kv8_batch *b, uint32_t qHeads) {
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

}  // namespace

extern "C" {

er_status er_hip_qk_norm_rope(er_hip_ctx *ctx, er_stream stream, const er_head_rows *q, const er_head_rows *k,
                              const er_head_rows *q_out, const er_head_rows *k_out, er_buffer positions,
                              er_buffer q_norm, er_buffer k_norm, const er_rope *rope, uint32_t rows,
                              uint32_t head_dim, float eps) {
    const char *op = "qk_norm_rope";
    er_status st = check_dim(op, head_dim);
    if (st == ER_OK) st = check_rope(op, rope, head_dim);
    if (st != ER_OK) return st;
    if (rows == 0) return check_ctx(ctx);
    if ((k == nullptr) != (k_out == nullptr))
        return fail(ER_ERR_INVALID_ARGUMENT, "%s: k and k_out come together", op);
    if (rows > 0x3fffffffu) return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u rows: over 2^30", op, rows);
    st = check_rows(op, "q", q, rows, head_dim, 4);
    if (st == ER_OK) st = check_rows(op, "q_out", q_out, rows, head_dim, 4);
    if (st == ER_OK && k) st = check_rows(op, "k", k, rows, head_dim, 4);
    if (st == ER_OK && k) st = check_rows(op, "k_out", k_out, rows, head_dim, 4);
    if (st != ER_OK) return st;
    if (q->heads != q_out->heads || (k && k->heads != k_out->heads))
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: outputs have other heads than inputs", op);
    st = check_apart(op, "q and q_out", q, q_out, rows, head_dim, 4, 4, true);
    if (st == ER_OK && k) st = check_apart(op, "k and k_out", k, k_out, rows, head_dim, 4, 4, true);
    if (st == ER_OK && k) st = check_apart(op, "q and k_out", q, k_out, rows, head_dim, 4, 4, false);
    if (st == ER_OK && k) st = check_apart(op, "k and q_out", k, q_out, rows, head_dim, 4, 4, false);
    if (st == ER_OK && k) st = check_apart(op, "q_out and k_out", q_out, k_out, rows, head_dim, 4, 4, false);
    if (st == ER_OK && rope->rotary_dim) st = check_buffer(op, "positions", positions, (uint64_t)rows * 4, 4);
    if (st == ER_OK) st = check_norm(op, "q_norm", q_norm, head_dim);
    if (st == ER_OK) st = check_norm(op, "k_norm", k_norm, head_dim);
    if (st == ER_OK) st = make_ready(op, ctx);
    if (st != ER_OK) return st;
    ErRopeArgs a{};
    a.q = turn_args(q, q_out, q_norm);
    if (k) a.k = turn_args(k, k_out, k_norm);
    a.positions = rope->rotary_dim ? (const int32_t *)positions.data : nullptr;
    a.freq = (const float *)rope->inv_freq.data;
    a.rot = rope->rotary_dim, a.pairs = rope->interleaved != 0;
    a.rows = rows, a.eps = eps;
    const uint32_t per = 512 / head_dim;
    a.chunks = row_chunks((a.q.heads + per - 1) / per + (a.k.heads + per - 1) / per, rows, cu_count_of(ctx));
    return launch(kv8_of(ctx).rope[dim_index(head_dim)], op, ((uint64_t)rows * a.chunks + 3) / 4, 0, stream, &a);
}

er_status er_hip_kv8_append(er_hip_ctx *ctx, er_stream stream, const er_kv8_cache *cache, const er_kv8_batch *batch,
                            const er_head_rows *k, const er_head_rows *v, uint32_t v_type, const er_head_rows *q,
                            const er_head_rows *q_out, er_buffer k_norm, er_buffer q_norm, const er_rope *rope,
                            float eps) {
    const char *op = "kv8_append";
    er_status st = check_cache(op, cache);
    if (st == ER_OK) st = check_rope(op, rope, cache->head_dim);
    if (st == ER_OK) st = check_batch(op, batch);
    if (st != ER_OK) return st;
    if (v_type != ER_TYPE_F32 && v_type != ER_TYPE_F16)
        return fail(ER_ERR_INVALID_ARGUMENT, "%s: v_type %u is not F32 or F16", op, v_type);
    if ((q == nullptr) != (q_out == nullptr))
        return fail(ER_ERR_INVALID_ARGUMENT, "%s: q and q_out come together", op);
    if (batch->rows == 0 || batch->sequences == 0) return check_ctx(ctx);
    const uint32_t d = cache->head_dim, vBytes = v_type == ER_TYPE_F16 ? 2 : 4;
    st = check_rows(op, "k", k, batch->rows, d, 4);
    if (st == ER_OK) st = check_rows(op, "v", v, batch->rows, d, vBytes);
    if (st == ER_OK && q) st = check_rows(op, "q", q, batch->rows, d, 4);
    if (st == ER_OK && q) st = check_rows(op, "q_out", q_out, batch->rows, d, 4);
    if (st != ER_OK) return st;
    if (k->heads != cache->kv_heads || v->heads != cache->kv_heads || (q && q->heads != q_out->heads))
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: k, v and cache, or q and q_out, differ in heads", op);
    if (q) {
        st = check_apart(op, "q and q_out", q, q_out, batch->rows, d, 4, 4, true);
        if (st == ER_OK) st = check_apart(op, "k and q_out", k, q_out, batch->rows, d, 4, 4, false);
        if (st == ER_OK) st = check_apart(op, "v and q_out", v, q_out, batch->rows, d, vBytes, 4, false);
    }
    if (st == ER_OK) st = check_norm(op, "k_norm", k_norm, d);
    if (st == ER_OK) st = check_norm(op, "q_norm", q_norm, d);
    if (st == ER_OK) st = make_ready(op, ctx);
    if (st != ER_OK) return st;
    ErAppendArgs a{};
    a.c = cache_args(cache), a.b = batch_args(cache, batch);
    a.k = (const float *)k->data.data, a.v = v->data.data;
    a.kNorm = (const float *)k_norm.data;
    a.kStride = k->row_stride, a.vStride = v->row_stride, a.vHalf = v_type == ER_TYPE_F16;
    a.freq = (const float *)rope->inv_freq.data;
    a.rot = rope->rotary_dim, a.pairs = rope->interleaved != 0;
    a.eps = eps;
    const uint32_t P = cache->page_tokens;
    // n tokens touch at most 1 + (n - 1 + P - 1) / P pages; no more than the table has
    a.spans = std::min((batch->max_rows + P - 2) / P + 1, std::max(1u, batch->table_stride));
    const uint64_t cacheBlocks = (uint64_t)batch->sequences * a.spans * cache->kv_heads * 2;
    uint64_t blocks = cacheBlocks;
    if (q) {
        a.q = turn_args(q, q_out, q_norm);
        const uint32_t per = 512 / d;
        a.chunks = row_chunks((a.q.heads + per - 1) / per, batch->rows, cu_count_of(ctx));
        blocks += ((uint64_t)batch->rows * a.chunks + 3) / 4;
    }
    st = check_blocks(op, blocks);
    if (st != ER_OK) return st;
    a.cacheBlocks = (uint32_t)cacheBlocks;
    return launch(kv8_of(ctx).append[dim_index(d)], op, blocks, 0, stream, &a);
}

er_status er_hip_kv8_attention_workspace(er_hip_ctx *ctx, const er_kv8_cache *cache, const er_kv8_batch *batch,
                                         uint32_t q_heads, uint64_t *bytes) {
    const char *op = "kv8_attention_workspace";
    if (!bytes) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null bytes", op);
    *bytes = 0;
    er_status st = check_cache(op, cache);
    if (st == ER_OK) st = check_batch(op, batch);
    if (st == ER_OK) st = check_group(op, cache, batch, q_heads);
    if (st == ER_OK) st = check_ctx(ctx);
    if (st != ER_OK) return st;
    if (batch->rows == 0 || batch->sequences == 0) return ER_OK;
    *bytes = plan_attend(cache, batch, q_heads / cache->kv_heads, 0, cu_count_of(ctx)).parts * (cache->head_dim + 2) * 4;
    return ER_OK;
}

er_status er_hip_kv8_attention(er_hip_ctx *ctx, er_stream stream, const er_kv8_cache *cache,
                               const er_kv8_batch *batch, const er_head_rows *q, const er_head_rows *out,
                               uint32_t out_type, float scale, uint32_t window, er_buffer workspace) {
    const char *op = "kv8_attention";
    er_status st = check_cache(op, cache);
    if (st == ER_OK) st = check_batch(op, batch);
    if (st != ER_OK) return st;
    if (out_type != ER_TYPE_F32 && out_type != ER_TYPE_BF16)
        return fail(ER_ERR_INVALID_ARGUMENT, "%s: out_type %u is not F32 or BF16", op, out_type);
    if (!std::isfinite(scale)) return fail(ER_ERR_INVALID_ARGUMENT, "%s: scale is not finite", op);
    if (batch->rows == 0 || batch->sequences == 0) return check_ctx(ctx);
    const uint32_t d = cache->head_dim, outBytes = out_type == ER_TYPE_BF16 ? 2 : 4;
    st = check_rows(op, "q", q, batch->rows, d, 4);
    if (st == ER_OK) st = check_rows(op, "out", out, batch->rows, d, outBytes);
    if (st != ER_OK) return st;
    if (q->heads != out->heads) return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: q and out differ in heads", op);
    st = check_group(op, cache, batch, q->heads);
    if (st == ER_OK) st = check_apart(op, "q and out", q, out, batch->rows, d, 4, outBytes, false);
    if (st == ER_OK) st = make_ready(op, ctx);
    if (st != ER_OK) return st;
    ErAttendArgs a{};
    a.c = cache_args(cache), a.b = batch_args(cache, batch);
    a.q = (const float *)q->data.data, a.out = out->data.data;
    a.qStride = q->row_stride, a.outStride = out->row_stride;
    a.group = q->heads / cache->kv_heads;
    a.window = window > 0x3fffffffu ? 0 : window;  // no sequence is as long
    a.half = out_type == ER_TYPE_BF16;
    a.scale = scale * 1.44269504088896340736f;
    const AttendPlan p = plan_attend(cache, batch, a.group, a.window, cu_count_of(ctx));
    a.shares = p.shares, a.least = p.least;
    a.splits = p.splits, a.chunk = p.chunk, a.tiles = p.tiles;
    const bool joined = p.splits > 1 || p.shares > 0;
    if (joined) {
        st = check_buffer(op, "workspace", workspace, p.parts * (d + 2) * 4, 16);
        if (st != ER_OK) return st;
        a.partO = (float *)workspace.data;
        a.partML = a.partO + p.parts * d;
    }
    const Kv8Kernels &kernels = kv8_of(ctx);
    const int di = dim_index(d);
    const uint64_t pairs = (uint64_t)batch->sequences * cache->kv_heads;
    const uint64_t blocks = p.shares ? p.shares : pairs * p.splits * p.tiles;  // narrow: one split
    const bool byRow = !p.shares && p.splits <= ER_KV8_ROW_PARTS;
    const uint64_t joins = !joined ? 0 : byRow ? batch->rows : (uint64_t)batch->rows * q->heads;
    // both, before the first is queued
    st = check_blocks(op, blocks);
    if (st == ER_OK) st = check_blocks(op, joins);
    if (st != ER_OK) return st;
    st = launch((p.narrow ? kernels.narrow : kernels.wide)[di][a.c.shift - 4][a.half], op, blocks, 0, stream, &a);
    if (st != ER_OK || !joined) return st;
    if (byRow) return launch(kernels.joinRow[di], op, joins, 0, stream, &a);
    const uint32_t most = p.shares ? p.shares : p.splits;
    return launch(kernels.join[di], op, joins, (4 * ER_KV8_THREADS + most) * 4, stream, &a);
}

}  // extern "C"
