// er_draft.cpp -- host side of what a step needs that drafts tokens, streams
// without end or answers under rules: attention under masks, acceptance of
// drafts, rules on logits.  Checks of arguments, launch plans, launches; nothing
// here allocates or synchronises, so every call can be recorded into a graph.
#include "er_draft.h"
#include "er_draft_host.h"
#include "er_kv8_check.h"

#include <cmath>
#include <cstdio>
#include <initializer_list>

extern "C" const unsigned char er_draft_blob[];

namespace er_detail {

er_status draft_load(DraftKernels &k) {
    hipError_t e = hipModuleLoadData(&k.module, er_draft_blob);
    if (e != hipSuccess) {
        k.module = nullptr;
        return fail(ER_ERR_LIBRARY_NOT_FOUND, "hipModuleLoadData(draft kernels): %s", hipGetErrorString(e));
    }
    static const int dims[kKv8Dims] = {64, 128, 256};
    static const char *const outs[2] = {"f32", "bf16"};
    er_status st = ER_OK;
    char name[64];
    auto find = [&](hipFunction_t &f, const char *form, auto... values) {
        if (st != ER_OK) return;
        std::snprintf(name, sizeof(name), form, values..., 0);
        const hipError_t r = hipModuleGetFunction(&f, k.module, name);
        if (r != hipSuccess) st = fail(ER_ERR_FUNCTION_NOT_FOUND, "functionNotFound(%s): %s", name, hipGetErrorString(r));
    };
    for (int d = 0; d < kKv8Dims; ++d) {
        for (int page = 0; page < kKv8Pages; ++page)
            for (int out = 0; out < 2; ++out) {
                for (int nb = 0; nb < 2; ++nb)
                    if (nb == 0 || dims[d] < 256)
                        find(k.few[nb][d][page][out], "er_kv8_masked_attend_c%d_d%d_p%d_%s", nb + 1, dims[d], 16 << page, outs[out]);
                find(k.wide[d][page][out], "er_kv8_masked_attend_wide_d%d_p%d_%s", dims[d], 16 << page, outs[out]);
            }
        for (int nb = 0; nb < (dims[d] < 256 ? 2 : 1); ++nb) {
            find(k.joinFew[nb][d], "er_kv8_masked_join_c%d_d%d", nb + 1, dims[d]);
            find(k.joinColumn[nb][d], "er_kv8_masked_join_column_c%d_d%d", nb + 1, dims[d]);
        }
        find(k.join[d], "er_kv8_masked_join_d%d", dims[d]);
        find(k.joinRow[d], "er_kv8_masked_join_row_d%d", dims[d]);
        find(k.accept[d], "er_kv8_accept_d%d", dims[d]);
    }
    for (int i = 0; i < 2; ++i) find(k.choose[i], "er_choose_s%d", 1 + i);
    find(k.chooseJoin, "er_choose_join");
    if (st != ER_OK) draft_unload(k);
    return st;
}

void draft_unload(DraftKernels &k) {
    if (k.module) (void)hipModuleUnload(k.module);
    k = DraftKernels{};
}

}  // namespace er_detail

namespace {

using namespace er_detail;

// The context's device current, its kernels there.
er_status make_ready(const char *op, const er_hip_ctx *ctx) {
    const er_status st = check_ctx(ctx);
    if (st != ER_OK) return st;
    if (!draft_of(ctx).module) return fail(ER_ERR_LIBRARY_NOT_FOUND, "%s: the draft kernels did not load with this context", op);
    return bind_device_of(ctx);
}

// Rows that are drafts, at most max_rows of each sequence, and their masks.
er_status check_drafts(const char *op, const er_drafts *d, uint32_t rows, uint32_t maxRows, bool masks) {
    if (maxRows > ER_MOST_DRAFTS)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u drafts of a sequence (at most %u)", op, maxRows, ER_MOST_DRAFTS);
    if (!masks) return ER_OK;
    if (d->seen_words > kMostHeads || (uint64_t)d->seen_words * 32 < maxRows)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u mask words a row for %u drafts", op, d->seen_words, maxRows);
    return check_buffer(op, "seen", d->seen, (uint64_t)rows * d->seen_words * 4, 4);
}

// How an attention call under masks is cut up: in shares as the narrow kernel's,
// with 16 or 32 columns a wave, or as the wide kernel's.
constexpr uint32_t kUnshared = 512;  // tokens of a sequence up to which a unit is never shared
uint32_t few_columns(const er_kv8_cache *c) { return c->head_dim == 256 ? 256 : 128; }
struct MaskedPlan : AttendPlan {
    uint32_t blocks;  // of 16 columns that a wave has; 0: the wide kernel
};
MaskedPlan plan_masked(const er_kv8_cache *c, const er_kv8_batch *b, uint32_t group, uint32_t window, int cu, uint32_t sinks,
                       bool drafts, bool half) {
    MaskedPlan p{};
    const uint64_t cols = (uint64_t)b->max_rows * group, full = most_tokens(c, b);
    // Shares against the wide kernel, us: trees of 128 columns of 32 sequences of up to 6000 tokens 149 / 196, of 192
    // of 8 of 4000 58 / 60, of 256 (bf16) 62 / 58, of 512 of 2 of 20000 122 / 107; of 256 of width 256 of 16 of 4000
    // 117 / 176.
    if (cols > few_columns(c)) {
        (AttendPlan &)p = plan_attend(c, b, group, window, cu, sinks, drafts);
        return p;
    }
    p.narrow = true;
    p.splits = 1;
    // 32 columns convert a tile's codes once for what 16 do twice, but leave half as many units, with twice as long a
    // start and end: taken where even so each share has some tiles.  16 / 32, us, by 64-token steps of 16 columns a
    // share: 1 (one user's tree) 13.8 / 16.5, 16 (three cases) 30.3 / 37.4, 29.8 / 32.4, 31.9 / 41.2, 170 (width 64)
    // 50.0 / 48.7, 390 214 / 149, 500 229 / 145.  At width 256 they do not fit: 117 / 133.
    const uint64_t steps = (uint64_t)b->sequences * c->kv_heads * ((cols + 15) / 16) * ((full + 63) / 64);
    p.blocks = c->head_dim < 256 && cols > 16 && steps >= 64ull * 2 * (uint64_t)cu ? 2 : 1;
    p.tiles = (uint32_t)((cols + 16 * p.blocks - 1) / (16 * p.blocks));
    // Where units are many and short, a workgroup has a unit each: shares cut some of them in two, whose sums a join then
    // reads, and a workgroup that goes from unit to unit waits for each one's lengths.  Shared / not, us, of sequences of
    // up to 1000 tokens (16 steps): 64 units 12.8 / 12.3, 96 15.2 / 12.5, 256 20.3 / 13.6 and 18.4 / 14.8, 512 34.2 / 20.0,
    // 1600 98 / 59; of 2000: 64 15.4 / 17.9, 128 17.6 / 18.0 and 20.5 / 19.2, 256 28.2 / 20.3, 512 51.9 / 38.9 and 32.9 /
    // 32.7; under a window of 2048: 512 64.2 / 54.1 and 46.0 / 36.1, 384 32.4 / 35.0; of 4000: 128 24.8 / 28.4, 256 44.9 /
    // 38.8, but 512 44.5 / 56.2, as the longest unit then decides.  At width 256 64 of 1000 17.6 / 24.5, 512 44.1 / 46.6.
    // The longest unit and their number do not tell all of these apart: the rule is wrong for 384 under the window (by 8%)
    // and for 256 of 4000 (by 16%).
    uint64_t span = full;
    if (window)
        span = std::min<uint64_t>(span, (uint64_t)window + b->max_rows + 127 + (((uint64_t)sinks + 63) & ~63ull));
    const uint64_t most = (span + 63) / 64, units = (uint64_t)b->sequences * c->kv_heads * p.tiles;
    const bool whole = c->head_dim < 256 && most <= 40 && units * 64 >= most * (uint64_t)cu && units <= kMostBlocks;
    if (span > kUnshared && !whole) {
        // Two workgroups a CU are resident; of the kernel whose registers leave a SIMD one wave (wide heads, two pages a
        // tile, two terms), one.  By one / two a CU, us: a user's 26 drafts behind 8000 tokens 25.3 / 33.6, 32 users' next
        // tokens behind 8000 69 / 82, trees of 100 of 8 of 4000 74.6 / 83.4, of 5 of 64 of 1000 29.5 / 37.7, of 5 of 8
        // of 2000 19.0 / 18.8.
        const bool one = c->head_dim == 256 && c->page_tokens == 16 && !half;
        p.shares = (uint32_t)cu * (one ? 1 : 2);
        p.parts = 4ull * (uint32_t)cu * 16 * p.blocks;  // of either output type
    }
    return p;
}

// The line that shares are cut from, with what rounds a unit's length up (fewer than 16 steps), is counted in 32 bits.
er_status check_line(const char *op, const er_kv8_cache *c, const er_kv8_batch *b, uint32_t group) {
    const uint64_t cols = (uint64_t)b->max_rows * group, full = most_tokens(c, b), steps = (full + 63) / 64 + 16;
    if (cols > few_columns(c) || full <= kUnshared || b->sequences * steps * c->kv_heads <= 0xffffffffull / ((cols + 15) / 16)) return ER_OK;
    return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u sequences of up to %u tokens and %u rows: too many to count in 32 bits", op,
                b->sequences, most_tokens(c, b), b->max_rows);
}

struct Range {
    const void *data;
    uint64_t bytes;
    const char *name;
};
// Outputs that no other buffer of the call may share memory with.
er_status check_no_overlap(const char *op, std::initializer_list<Range> outputs, std::initializer_list<Range> inputs) {
    auto meet = [&](const Range &a, const Range &b) {
        const uintptr_t x = (uintptr_t)a.data, y = (uintptr_t)b.data;
        return a.data && b.data && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
    };
    for (const Range *a = outputs.begin(); a != outputs.end(); ++a) {
        for (const Range *b = a + 1; b != outputs.end(); ++b)
            if (meet(*a, *b)) return fail(ER_ERR_INVALID_ARGUMENT, "%s: %s and %s overlap", op, a->name, b->name);
        for (const Range &b : inputs)
            if (meet(*a, b)) return fail(ER_ERR_INVALID_ARGUMENT, "%s: %s and %s overlap", op, a->name, b.name);
    }
    return ER_OK;
}

// Tokens of a row that one workgroup takes.  Few of them scan the context more often, many have room in LDS for fewer
// workgroups at once: by 1024, 2048, 4096, us, one user 7.5, 7.5, 8.7, 64 users with 4096 tokens of context, biases and
// masks 29.6, 23.9, 32.8, 172 nodes of trees 57, 42, 46.  A vocabulary below a slice takes half.
struct ChoosePlan {
    uint32_t slices, slice;
};
ChoosePlan plan_choose(uint32_t vocab) {
    const uint32_t slice = vocab < ER_CHOOSE_SLICE ? ER_CHOOSE_SLICE / 2 : ER_CHOOSE_SLICE;
    return ChoosePlan{(vocab + slice - 1) / slice, slice};
}
uint64_t choose_workspace(uint32_t rows, uint32_t vocab) { return (uint64_t)rows * plan_choose(vocab).slices * 8; }

er_status check_logits(const char *op, uint32_t rows, uint32_t vocab) {
    if (rows > 0x3fffffffu || vocab == 0 || vocab > 0x3fffffffu)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u rows of %u logits", op, rows, vocab);
    return ER_OK;
}

// A list of each sequence's: values, their counts, entries a sequence may have.
er_status check_list(const char *op, const char *what, const er_buffer &values, uint32_t stride, uint32_t sequences) {
    if (stride > 0x3fffffffu) return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %s of %u entries a sequence", op, what, stride);
    return check_buffer(op, what, values, (uint64_t)sequences * stride * 4, 4);
}

}  // namespace

extern "C" {

er_status er_hip_kv8_attention_masked(er_hip_ctx *ctx, er_stream stream, const er_kv8_cache *cache,
                                      const er_kv8_batch *batch, const er_head_rows *q, const er_head_rows *out,
                                      uint32_t out_type, float scale, uint32_t window, uint32_t sinks,
                                      const er_drafts *drafts, er_buffer workspace) {
    const char *op = "kv8_attention_masked";
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
    if (st == ER_OK) st = check_line(op, cache, batch, q->heads / cache->kv_heads);
    if (st == ER_OK) st = check_apart(op, "q and out", q, out, batch->rows, d, 4, outBytes, false);
    if (st == ER_OK && drafts) st = check_drafts(op, drafts, batch->rows, batch->max_rows, true);
    if (st == ER_OK && drafts && window) st = check_buffer(op, "position", drafts->position, (uint64_t)batch->rows * 4, 4);
    if (st == ER_OK) st = make_ready(op, ctx);
    if (st != ER_OK) return st;
    ErMaskedArgs a{};
    a.c = cache_args(cache), a.b = batch_args(cache, batch);
    a.q = (const float *)q->data.data, a.out = out->data.data;
    a.qStride = q->row_stride, a.outStride = out->row_stride;
    a.group = q->heads / cache->kv_heads;
    a.window = window > 0x3fffffffu ? 0 : window;  // no sequence is as long
    a.sinks = std::min(sinks, 0x3fffffffu);
    a.half = out_type == ER_TYPE_BF16;
    a.scale = scale * 1.44269504088896340736f;
    if (drafts) {
        a.seen = (const uint32_t *)drafts->seen.data;
        a.words = drafts->seen_words;
        a.position = (const int32_t *)drafts->position.data;
    }
    const MaskedPlan p = plan_masked(cache, batch, a.group, a.window, cu_count_of(ctx), a.sinks, drafts != nullptr, a.half);
    a.shares = p.shares;
    a.splits = p.splits, a.chunk = p.chunk, a.tiles = p.tiles;
    const DraftKernels &kernels = draft_of(ctx);
    const int di = dim_index(d), nb = (int)p.blocks - 1;
    if (p.blocks == 0)
        return launch_attend(op, kernels.wide[di][a.c.shift - 4][a.half],
                             join_of(p, kernels.join[di], kernels.joinRow[di], batch->rows, q->heads), a, p, d, workspace, stream);
    // A workgroup a column where the chip holds as many at once (8 a CU); else one for some of a row's heads.  By
    // columns, us: 416 13.8 / 19.9, 512 29.8 / 45.3, 832 35.8 / 43.2, 1536 149 / 151, 2560 30.9 / 30.3, 6720 59 / 50
    const uint32_t together = ER_KV8_THREADS / (d / 4);
    JoinLaunch join = join_of(p, kernels.joinColumn[nb][di], nullptr, batch->rows, q->heads);
    if (join.blocks > 8ull * (uint64_t)cu_count_of(ctx))
        join = JoinLaunch{kernels.joinFew[nb][di], (uint64_t)batch->rows * ((q->heads + together - 1) / together), 0};
    return launch_attend(op, kernels.few[nb][di][a.c.shift - 4][a.half], join, a, p, d, workspace, stream);
}

er_status er_hip_kv8_attention_masked_workspace(er_hip_ctx *ctx, const er_kv8_cache *cache, const er_kv8_batch *batch,
                                                uint32_t q_heads, uint64_t *bytes) {
    const char *op = "kv8_attention_masked_workspace";
    if (!bytes) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null bytes", op);
    *bytes = 0;
    er_status st = check_cache(op, cache);
    if (st == ER_OK) st = check_batch(op, batch);
    if (st == ER_OK) st = check_group(op, cache, batch, q_heads);
    if (st == ER_OK) st = check_line(op, cache, batch, q_heads / cache->kv_heads);
    if (st == ER_OK) st = check_ctx(ctx);
    if (st != ER_OK) return st;
    if (batch->rows == 0 || batch->sequences == 0) return ER_OK;
    const MaskedPlan p = plan_masked(cache, batch, q_heads / cache->kv_heads, 0, cu_count_of(ctx), 0, false, false);
    *bytes = p.parts * (cache->head_dim + 2) * 4;
    return ER_OK;
}

er_status er_hip_kv8_accept(er_hip_ctx *ctx, er_stream stream, const er_kv8_cache *cache, const er_kv8_batch *batch,
                            const er_drafts *drafts, er_buffer chosen, er_buffer path, er_buffer count, er_buffer next,
                            er_buffer kv_len) {
    const char *op = "kv8_accept";
    er_status st = check_cache(op, cache);
    if (st == ER_OK) st = check_batch(op, batch);
    if (st != ER_OK) return st;
    if (!drafts) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null drafts", op);
    const uint64_t seqs = (uint64_t)batch->sequences * 4, rows = (uint64_t)batch->rows * 4;
    const uint64_t blocks = (uint64_t)cache->pages * cache->kv_heads, codes = (uint64_t)cache->page_tokens * cache->head_dim;
    if (batch->sequences == 0) return check_ctx(ctx);
    if (batch->rows == 0) {
        // what sequences without rows have is written all the same, and check_batch has not looked at what that reads
        st = check_buffer(op, "kv_len", batch->kv_len, seqs, 4);
        if (st == ER_OK) st = check_buffer(op, "row_start", batch->row_start, seqs + 4, 4);
    } else {
        st = check_drafts(op, drafts, batch->rows, batch->max_rows, false);
        if (st == ER_OK) st = check_buffer(op, "parent", drafts->parent, rows, 4);
        if (st == ER_OK) st = check_buffer(op, "token", drafts->token, rows, 4);
        if (st == ER_OK) st = check_buffer(op, "chosen", chosen, rows, 4);
        if (st == ER_OK) st = check_buffer(op, "path", path, rows, 4);
    }
    if (st == ER_OK) st = check_buffer(op, "count", count, seqs, 4);
    if (st == ER_OK) st = check_buffer(op, "next", next, seqs, 4);
    if (st == ER_OK) st = check_buffer(op, "kv_len", kv_len, seqs, 4);
    if (st == ER_OK)
        // every workgroup of a sequence reads the arrays that the first one's results stand beside
        st = check_no_overlap(op, {{path.data, rows, "path"}, {count.data, seqs, "count"}, {next.data, seqs, "next"},
                                   {kv_len.data, seqs, "kv_len"}},
                              {{drafts->parent.data, rows, "parent"}, {drafts->token.data, rows, "token"},
                               {chosen.data, rows, "chosen"}, {batch->kv_len.data, seqs, "the batch's kv_len"},
                               {batch->row_start.data, seqs + 4, "row_start"},
                               {batch->page_table.data, seqs * batch->table_stride, "the page table"},
                               {cache->k.data, blocks * codes, "k cache"}, {cache->v.data, blocks * codes, "v cache"},
                               {cache->k_scale.data, blocks * 4, "k scales"}, {cache->v_scale.data, blocks * 4, "v scales"}});
    if (st == ER_OK) st = make_ready(op, ctx);
    if (st != ER_OK) return st;
    ErAcceptArgs a{};
    a.c = cache_args(cache), a.b = batch_args(cache, batch);
    a.parent = (const int32_t *)drafts->parent.data, a.token = (const int32_t *)drafts->token.data;
    a.chosen = (const int32_t *)chosen.data;
    a.path = (int32_t *)path.data, a.count = (int32_t *)count.data;
    a.next = (int32_t *)next.data, a.left = (int32_t *)kv_len.data;
    return launch(draft_of(ctx).accept[dim_index(cache->head_dim)], op, (uint64_t)batch->sequences * cache->kv_heads * 2, 0,
                  stream, &a);
}

er_status er_hip_choose_logits_workspace(er_hip_ctx *ctx, uint32_t rows, uint32_t vocab, uint64_t *bytes) {
    const char *op = "choose_logits_workspace";
    if (!bytes) return fail(ER_ERR_INVALID_ARGUMENT, "%s: null bytes", op);
    *bytes = 0;
    er_status st = check_logits(op, rows, vocab);
    if (st == ER_OK) st = check_ctx(ctx);
    if (st != ER_OK) return st;
    *bytes = choose_workspace(rows, vocab);
    return ER_OK;
}

er_status er_hip_choose_logits(er_hip_ctx *ctx, er_stream stream, er_buffer logits, uint32_t rows, uint32_t vocab,
                               uint32_t row_stride, const er_logit_rules *rules, const er_drafts *drafts, er_buffer out,
                               er_buffer chosen, er_buffer workspace) {
    const char *op = "choose_logits";
    er_status st = check_logits(op, rows, vocab);
    if (st != ER_OK) return st;
    if (row_stride < vocab || row_stride > 0x3fffffffu)
        return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: row stride %u for %u logits", op, row_stride, vocab);
    if (!out.data && !chosen.data) return fail(ER_ERR_INVALID_ARGUMENT, "%s: neither out nor chosen", op);
    if (rows == 0) return check_ctx(ctx);
    const uint64_t span = ((uint64_t)(rows - 1) * row_stride + vocab) * 4, need = choose_workspace(rows, vocab);
    st = check_buffer(op, "logits", logits, span, 4);
    if (st == ER_OK && out.data) st = check_buffer(op, "out", out, span, 4);
    if (st == ER_OK && chosen.data) st = check_buffer(op, "chosen", chosen, (uint64_t)rows * 4, 4);
    if (st == ER_OK && chosen.data) st = check_buffer(op, "workspace", workspace, need, 4);
    if (st != ER_OK) return st;
    ErChooseArgs a{};
    a.logits = (const float *)logits.data, a.out = (float *)out.data, a.chosen = (int32_t *)chosen.data;
    a.rows = rows, a.vocab = vocab, a.stride = row_stride;
    a.sequences = rows, a.maxRows = 1;
    const uint64_t words = ((uint64_t)vocab + 31) / 32;
    uint64_t seqs = 0, allowed = 0;
    if (rules) {
        const er_logit_rules &r = *rules;
        if (r.row_start.data) {
            if (r.sequences == 0) return check_ctx(ctx);
            if (r.sequences > 0x3fffffffu || r.max_rows == 0 || r.max_rows > rows)
                return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u sequences, max_rows %u of %u rows", op, r.sequences, r.max_rows, rows);
            st = check_buffer(op, "row_start", r.row_start, ((uint64_t)r.sequences + 1) * 4, 4);
            a.start = (const int32_t *)r.row_start.data;
            a.sequences = r.sequences, a.maxRows = r.max_rows;
        }
        seqs = (uint64_t)a.sequences * 4;
        if (st == ER_OK && r.penalty.data) st = check_buffer(op, "penalty", r.penalty, seqs * 3, 4);
        if (st == ER_OK && r.history.data) st = check_list(op, "history", r.history, r.history_stride, a.sequences);
        if (st == ER_OK && r.history.data) st = check_buffer(op, "history_len", r.history_len, seqs, 4);
        if (st == ER_OK && r.bias.data) st = check_list(op, "bias", r.bias, r.bias_stride, a.sequences);
        if (st == ER_OK && r.bias.data) st = check_list(op, "bias_token", r.bias_token, r.bias_stride, a.sequences);
        if (st == ER_OK && r.bias.data) st = check_buffer(op, "bias_len", r.bias_len, seqs, 4);
        if (st == ER_OK && r.allowed.data) {
            if (r.allowed_stride < words)
                return fail(ER_ERR_INVALID_VECTOR_SHAPE, "%s: %u mask words a row for %u logits", op, r.allowed_stride, vocab);
            allowed = ((uint64_t)(rows - 1) * r.allowed_stride + words) * 4;
            st = check_buffer(op, "allowed", r.allowed, allowed, 4);
        }
        if (st != ER_OK) return st;
        a.penalty = (const float *)r.penalty.data;
        a.history = (const int32_t *)r.history.data, a.historyLen = (const int32_t *)r.history_len.data;
        a.historyStride = r.history_stride;
        a.bias = (const float *)r.bias.data, a.biasToken = (const int32_t *)r.bias_token.data;
        a.biasLen = (const int32_t *)r.bias_len.data, a.biasStride = r.bias_stride;
        a.allowed = (const uint32_t *)r.allowed.data, a.allowedStride = r.allowed_stride;
    }
    if (drafts) {
        st = check_drafts(op, drafts, rows, a.maxRows, true);
        if (st == ER_OK) st = check_buffer(op, "token", drafts->token, (uint64_t)rows * 4, 4);
        if (st != ER_OK) return st;
        a.seen = (const uint32_t *)drafts->seen.data, a.words = drafts->seen_words;
        a.token = (const int32_t *)drafts->token.data;
    }
    const bool inPlace = out.data == logits.data;
    const uint64_t parts = chosen.data ? need : 0, lists = seqs * a.historyStride, biases = seqs * a.biasStride;
    st = check_no_overlap(op, {{out.data, span, "out"}, {chosen.data, (uint64_t)rows * 4, "chosen"}, {workspace.data, parts, "workspace"}},
                          {{inPlace ? nullptr : logits.data, span, "logits"}, {a.start, seqs + 4, "row_start"},
                           {a.penalty, seqs * 3, "penalty"}, {a.history, lists, "history"}, {a.historyLen, seqs, "history_len"},
                           {a.bias, biases, "bias"}, {a.biasToken, biases, "bias_token"}, {a.biasLen, seqs, "bias_len"},
                           {a.allowed, allowed, "allowed"}, {a.seen, (uint64_t)rows * a.words * 4, "seen"},
                           {a.token, (uint64_t)rows * 4, "token"}});
    if (st == ER_OK && inPlace)
        st = check_no_overlap(op, {{chosen.data, (uint64_t)rows * 4, "chosen"}, {workspace.data, parts, "workspace"}},
                              {{logits.data, span, "logits"}});
    if (st == ER_OK) st = make_ready(op, ctx);
    if (st != ER_OK) return st;
    const ChoosePlan plan = plan_choose(vocab);
    a.slices = plan.slices;
    a.partV = (float *)workspace.data;
    a.partI = (uint32_t *)workspace.data + (uint64_t)rows * plan.slices;
    // counts, entries and the list
    const uint32_t lds = a.penalty || a.bias ? plan.slice * (a.bias ? 10 : 6) : 0;
    const uint64_t blocks = (uint64_t)rows * plan.slices, joins = ((uint64_t)rows + 3) / 4;
    st = check_blocks(op, blocks);
    if (st == ER_OK) st = launch(draft_of(ctx).choose[plan.slice < ER_CHOOSE_SLICE ? 0 : 1], op, blocks, lds, stream, &a);
    if (st != ER_OK || !chosen.data || plan.slices == 1) return st;
    return launch(draft_of(ctx).chooseJoin, op, joins, 0, stream, &a);
}

}  // extern "C"
