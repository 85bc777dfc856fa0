// er_kv8.cpp -- host side of the operators between the projections (head norms
// with the rotation, the 8-bit paged cache, attention over it): checks of
// arguments, launch plans, launches.  Nothing here allocates or synchronises,
// so every call can be recorded into a graph.
#include "er_hip.h"
#include "er_kv8_check.h"

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

ErTurn turn_args(const er_head_rows *in, const er_head_rows *out, const er_buffer &norm) {
    ErTurn t{};
    t.in = (const float *)in->data.data, t.out = (float *)out->data.data;
    t.norm = (const float *)norm.data;
    t.inStride = in->row_stride, t.outStride = out->row_stride, t.heads = in->heads;
    return t;
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
    const Kv8Kernels &kernels = kv8_of(ctx);
    const int di = dim_index(d);
    return launch_attend(op, (p.narrow ? kernels.narrow : kernels.wide)[di][a.c.shift - 4][a.half],
                         join_of(p, kernels.join[di], kernels.joinRow[di], batch->rows, q->heads), a, p, d, workspace, stream);
}

}  // extern "C"
