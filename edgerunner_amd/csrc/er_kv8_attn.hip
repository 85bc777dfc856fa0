// er_kv8_attn.hip -- attention over the 8-bit paged cache (part of er_kv8.hip).
//
// Columns are (row, query head) pairs of one sequence that share a key/value
// head.  Both kernels form S^T = K Q^T (keys down, columns across) on the
// matrix cores, whose output gives a lane one column: the softmax's running
// maximum and sum are plain values of the lane, and the weights, rounded to
// fp16, are already the second product's B operand, O^T = V^T W^T, if V's
// tokens are taken in the order in which S^T's rows lie in the lanes.  No
// weight crosses lanes.
//
// e4m3 codes are exact in fp16 (11 bits), so codes go to the matrix cores as
// they are: a key block's scale multiplies the scores, a value block's scale,
// over the largest seen so far, enters with the code's conversion.  For fp32
// output the query and the weights are split into two fp16 terms (22 bits) and
// the products formed twice; for bf16 output one term (11 bits, to bf16's 8)
// does.  Sums, maxima and outputs are fp32 throughout.
//
// The running maximum is a reference that only moves when a score passes it
// by more than 8 (in powers of two); weights are 2^(s - m + 7), so at most
// 2^15, and the reference cancels in the quotient.  Most tiles rescale nothing.

#define ER_NO_MAX (-1.0e30f)  // reference of a column that has seen no score

ER_DEV f32x4 mfma16(h8 a, h8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
ER_DEV f32x16 mfma32(h8 a, h8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Two of a dword's four codes (low or high half) as fp16, times a power of two.
template <bool HIGH>
ER_DEV h2 codes_to_h2(uint32_t c, float f) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, f, HIGH);
}
ER_DEV h8 join(h2 a, h2 b, h2 c, h2 d) { return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}; }
ER_DEV h8 codes_to_h8(uint32_t lo, uint32_t hi) {
    return join(codes_to_h2<false>(lo, 1.0f), codes_to_h2<true>(lo, 1.0f), codes_to_h2<false>(hi, 1.0f),
                codes_to_h2<true>(hi, 1.0f));
}
// Bytes (x0 x1 x2 x3), (y0 y1 y2 y3) to (x0 y0 x1 y1) and (x2 y2 x3 y3).
ER_DEV uint32_t zip_lo(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x05010400u); }
ER_DEV uint32_t zip_hi(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07030602u); }

// Four codes each of eight tokens (dword w of each) to four A operands, one a
// code, of the eight tokens; f0 scales the first four tokens, f1 the others.
ER_DEV void transpose_codes(const uint32_t x[8], float f0, float f1, h8 out[4]) {
    const uint32_t a0 = zip_lo(x[0], x[1]), a1 = zip_hi(x[0], x[1]), b0 = zip_lo(x[2], x[3]), b1 = zip_hi(x[2], x[3]);
    const uint32_t c0 = zip_lo(x[4], x[5]), c1 = zip_hi(x[4], x[5]), d0 = zip_lo(x[6], x[7]), d1 = zip_hi(x[6], x[7]);
    out[0] = join(codes_to_h2<false>(a0, f0), codes_to_h2<false>(b0, f0), codes_to_h2<false>(c0, f1), codes_to_h2<false>(d0, f1));
    out[1] = join(codes_to_h2<true>(a0, f0), codes_to_h2<true>(b0, f0), codes_to_h2<true>(c0, f1), codes_to_h2<true>(d0, f1));
    out[2] = join(codes_to_h2<false>(a1, f0), codes_to_h2<false>(b1, f0), codes_to_h2<false>(c1, f1), codes_to_h2<false>(d1, f1));
    out[3] = join(codes_to_h2<true>(a1, f0), codes_to_h2<true>(b1, f0), codes_to_h2<true>(c1, f1), codes_to_h2<true>(d1, f1));
}

// The NaN codes of an operand: is there one, ones in their places, zeros in their places.
ER_DEV bool is_nan_h(_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7fffu) > 0x7c00u; }
ER_DEV bool any_nan(h8 x) {
    bool n = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) n |= is_nan_h(x[i]);
    return n;
}
ER_DEV h8 nan_places(h8 x) {
    h8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = is_nan_h(x[i]) ? (_Float16)1.0f : (_Float16)0.0f;
    return r;
}
ER_DEV h8 without_nan(h8 x) {
    h8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = is_nan_h(x[i]) ? (_Float16)0.0f : x[i];
    return r;
}

// A column of a tile: its row, its query head, and the tokens [lo, hi) that it sees.
struct Column {
    int row, lo, hi;
    uint32_t head;
};
ER_DEV Column column_of(const ErAttendArgs &p, const Sequence &q, uint32_t kvHead, uint32_t col) {
    Column c;
    const uint32_t r = col / p.group;
    const int pos = q.len - q.n + (int)r;
    c.row = q.row0 + (int)r;
    c.head = kvHead * p.group + (col - r * p.group);
    c.hi = max(pos + 1, 0);
    c.lo = p.window && c.hi > (int)p.window ? c.hi - (int)p.window : 0;
    return c;
}

// A column's query as B operands: eight consecutive values from `from` on for
// each of N products, `step` values apart, as one or two fp16 terms.  The
// query is brought to below 1 by a power of two over the whole head (`join`
// takes the largest magnitude over the lanes that share the column); returns
// that power.
template <int N, int TERMS, typename JOIN>
ER_DEV float load_query(const float *src, bool live, uint32_t from, uint32_t step, h8 (&b)[TERMS][N], JOIN join_lanes) {
    float x[N][8];
    float peak = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        f32x4 lo = {}, hi = {};
        if (live) {
            lo = *(const f32x4_a4 *)(src + from + k * step);
            hi = *(const f32x4_a4 *)(src + from + k * step + 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[k][i] = lo[i];
            x[k][4 + i] = hi[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) peak = fmaxf(peak, finite_magnitude(x[k][i]));
    }
    peak = join_lanes(peak);
    // peak < 2^e; e stays where 2^-e is a normal number
    const int e = min(max((int)(__float_as_uint(peak) >> 23) - 126, -126), 126);
    const float f = exp2i(-e);
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = x[k][i] * f;
            const _Float16 h = (_Float16)v;
            b[0][k][i] = h;
            if constexpr (TERMS == 2) b[1][k][i] = (_Float16)(v - (float)h);
        }
    return exp2i(e);
}

// Weights of eight tokens as one or two fp16 terms.
template <int TERMS>
ER_DEV void weight_terms(const float w[8], h8 (&b)[TERMS]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const _Float16 h = (_Float16)w[i];
        b[0][i] = h;
        if constexpr (TERMS == 2) b[1][i] = (_Float16)(w[i] - (float)h);
    }
}

ER_DEV uint16_t to_bf16(float v) {  // nearest even; a NaN stays one
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
ER_DEV void store4(const ErAttendArgs &p, int row, uint32_t head, uint32_t d, uint32_t D, f32x4 v) {
    const size_t at = (size_t)row * p.outStride + (size_t)head * D + d;
    if (p.half)
        *(u16x4_a2 *)((uint16_t *)p.out + at) = u16x4_a2{to_bf16(v.x), to_bf16(v.y), to_bf16(v.z), to_bf16(v.w)};
    else
        *(f32x4_a4 *)((float *)p.out + at) = v;
}
// Index of a column's partial sums of one piece.
ER_DEV size_t part_index(const ErAttendArgs &p, uint32_t piece, int row, uint32_t head) {
    return ((size_t)piece * p.b.rows + (size_t)row) * (p.group * p.c.heads) + head;
}
// sum / weight; zeros where no token is visible.  Where some are and the sum
// of weights is 0 or NaN (scores without a finite maximum), the quotient is
// NaN, as the softmax's is.
ER_DEV float quotient(float l, bool visible) { return visible ? 1.0f / l : 0.0f; }

// ---------------------------------------------------------------- up to 16 columns: decode

// One 32-token tile of keys and values in registers, as loaded.
template <int D>
struct NarrowTile {
    u32x4 k[2][D / 64];      // lane (n, g): token n of each half, bytes [g D/4, (g + 1) D/4)
    uint32_t v[D / 64][8];   // lane (n, g): tokens 4 g + i of the first half, then of the second, bytes [n D/16, (n + 1) D/16)
    float ks[2], vs[2];      // the halves' scales
    bool ok[2];              // the half's page exists and holds a visible token
};

template <int D>
ER_DEV void load_narrow(NarrowTile<D> &t, const ErAttendArgs &p, uint32_t s, uint32_t h, int T, int lo, int hi,
                        uint32_t n, uint32_t g) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int at = T + 16 * half;
        int page = -1;
        if (at < hi && at + 16 > lo) page = uniform(page_of(p.b, p.c, s, at));
        t.ok[half] = page >= 0;
        const size_t block = (size_t)(uint32_t)max(page, 0) * p.c.heads + h;
        t.ks[half] = p.c.ks[block];
        t.vs[half] = p.c.vs[block];
        const uint32_t inside = (uint32_t)at & ((1u << p.c.shift) - 1u);
        const size_t base = ((block << p.c.shift) + inside) * D;
        const uint8_t *kp = p.c.k + base + n * D + g * (D / 4);
        const uint8_t *vp = p.c.v + base + 4 * g * D + n * (D / 16);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) t.k[half][j] = *(const u32x4 *)(kp + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (D == 64) {
                t.v[0][4 * half + i] = *(const uint32_t *)(vp + i * D);
            } else if constexpr (D == 128) {
                const u32x2 w = *(const u32x2 *)(vp + i * D);
                t.v[0][4 * half + i] = w.x;
                t.v[1][4 * half + i] = w.y;
            } else {
                const u32x4 w = *(const u32x4 *)(vp + i * D);
                t.v[0][4 * half + i] = w.x;
                t.v[1][4 * half + i] = w.y;
                t.v[2][4 * half + i] = w.z;
                t.v[3][4 * half + i] = w.w;
            }
        }
    }
}

// The largest value over the four lanes n, n + 16, n + 32, n + 48.
ER_DEV float column_max4(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
ER_DEV float column_sum4(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Running state of a wave's 16 columns.
template <int D>
struct NarrowState {
    f32x4 o[D / 16];  // o[j][i]: value (4 g + i) D/16 + j of column n
    float m, l;       // reference; this lane's part of the sum of weights
    float vref;       // the largest value scale so far: o is in units of vref / 128 (wave-uniform)
    bool seen;        // a token was visible to the column
};

// Tokens that some column sees, and tokens that every column sees.
struct Spans {
    int anyLo, anyHi, allLo, allHi;
};
ER_DEV Spans spans_of(const ErAttendArgs &p, const Sequence &q, uint32_t firstCol, uint32_t lastCol) {
    const Column a = column_of(p, q, 0, firstCol), b = column_of(p, q, 0, lastCol);
    return Spans{a.lo, b.hi, b.lo, a.hi};
}

// One product of the values with the weights, where a tile that the columns
// see in part holds NaN codes: a token hidden from a column must leave it
// alone, and 0 * NaN would not.  The NaN codes count as zeros, and a second
// product counts the visible ones.
template <int TERMS>
ER_DEV void add_values(f32x4 &o, h8 a, const h8 (&b)[TERMS], h8 visible, bool nans) {
    if (!nans) {
#pragma unroll
        for (int term = 0; term < TERMS; ++term) o = mfma16(a, b[term], o);
        return;
    }
    const f32x4 hits = mfma16(nan_places(a), visible, f32x4{});
    a = without_nan(a);
#pragma unroll
    for (int term = 0; term < TERMS; ++term) o = mfma16(a, b[term], o);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = hits[i] > 0.0f ? __builtin_nanf("") : o[i];
}

template <int D, int TERMS>
ER_DEV void attend_narrow(NarrowState<D> &st, const NarrowTile<D> &t, const h8 (&qb)[TERMS][D / 32], float qf, int T,
                          int lo, int hi, const Spans &w, uint32_t g) {
    if (!t.ok[0] && !t.ok[1]) return;
    float x[8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        f32x4 s = {};
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const u32x4 c = t.k[half][k / 2];
            const h8 a = k % 2 ? codes_to_h8(c.z, c.w) : codes_to_h8(c.x, c.y);
#pragma unroll
            for (int term = 0; term < TERMS; ++term) s = mfma16(a, qb[term][k], s);
        }
        const float f = qf * t.ks[half];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * half + i] = s[i] * f;
    }
    const bool whole = t.ok[0] && t.ok[1] && T >= w.allLo && T + 32 <= w.allHi;
    uint32_t shown = 0xff;
    if (!whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int tok = T + 16 * (i / 4) + 4 * (int)g + (i & 3);
            if (!(t.ok[i / 4] && tok >= lo && tok < hi)) {
                x[i] = -__builtin_inff();
                shown &= ~(1u << i);
            }
        }
    }
    st.seen |= shown != 0;
    const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (__any(top > st.m + 8.0f)) {
        const float m = fmaxf(st.m, column_max4(top));
        const float f = __builtin_amdgcn_exp2f(st.m - m);
        st.m = m;
        st.l *= f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st.o[j] *= f;
    }
    const float vs0 = t.ok[0] ? t.vs[0] : t.vs[1], vs1 = t.ok[1] ? t.vs[1] : t.vs[0];
    const float vtop = fmaxf(vs0, vs1);
    if (vtop > st.vref) {
        const float f = st.vref / vtop;
        st.vref = vtop;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st.o[j] *= f;
    }
    const float f0 = 128.0f * (vs0 / st.vref), f1 = 128.0f * (vs1 / st.vref);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_amdgcn_exp2f(x[i] - (st.m - 7.0f));
        st.l += x[i];
    }
    h8 b[TERMS], visible;
    weight_terms<TERMS>(x, b);
    // whole tiles, and those whose hidden tokens are hidden from all columns, need no care with NaN codes
    const bool mixed = !whole && (w.anyLo < w.allLo || w.anyHi > w.allHi);
#pragma unroll
    for (int i = 0; i < 8; ++i) visible[i] = (shown >> i) & 1u ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = t.v[d][i];
        if (!whole) {
            // tokens that no column sees, or without a page, count as zeros whatever their bytes hold
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int tok = T + 16 * (i / 4) + 4 * (int)g + (i & 3);
                c[i] = t.ok[i / 4] && tok >= w.anyLo && tok < w.anyHi ? c[i] : 0u;
            }
        }
        h8 a[4];
        transpose_codes(c, f0, f1, a);
        const bool nans = mixed && __any(any_nan(a[0]) || any_nan(a[1]) || any_nan(a[2]) || any_nan(a[3]));
#pragma unroll
        for (int j = 0; j < 4; ++j) add_values<TERMS>(st.o[4 * d + j], a[j], b, visible, nans);
    }
}

// Up to 16 columns (rows of one sequence times query heads of one key/value
// head) against one piece of its tokens: bound by the bytes of the cache.
// Every wave takes each fourth 32-token tile straight into registers, 8 KB of
// codes at head width 128, with the next tile in flight while it works; keys
// and values need no exchange between lanes, so nothing passes through LDS
// until the waves' sums are joined at the end.
template <int D, int TERMS>
ER_DEV void kv8_attend_narrow(const ErAttendArgs &p, float *lds) {
    const uint32_t piece = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
    const uint32_t h = unit % p.c.heads, s = unit / p.c.heads;
    const Sequence q = sequence_of(p.b, s);
    if (q.n == 0) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), n = lane & 15u, g = lane >> 4;
    const uint32_t cols = (uint32_t)q.n * p.group;
    const Spans w = spans_of(p, q, 0, cols - 1);
    const int begin = (w.anyLo & ~63) + (int)(piece * p.chunk), end = min(w.anyHi, begin + (int)p.chunk);
    const Column c = column_of(p, q, h, min(n, cols - 1));

    NarrowTile<D> t0, t1;
    int T = begin + 32 * (int)wave;
    if (T < end) load_narrow<D>(t0, p, s, h, T, w.anyLo, end, n, g);
    h8 qb[TERMS][D / 32];
    const float qf = load_query<D / 32, TERMS>(p.q + (size_t)c.row * p.qStride + (size_t)c.head * D, n < cols,
                                               g * (D / 4), 8, qb, column_max4) * p.scale;
    NarrowState<D> st = {};
    st.m = ER_NO_MAX;
    while (T < end) {
        if (T + 128 < end) load_narrow<D>(t1, p, s, h, T + 128, w.anyLo, end, n, g);
        attend_narrow<D, TERMS>(st, t0, qb, qf, T, c.lo, c.hi, w, g);
        T += 128;
        if (T >= end) break;
        if (T + 128 < end) load_narrow<D>(t0, p, s, h, T + 128, w.anyLo, end, n, g);
        attend_narrow<D, TERMS>(st, t1, qb, qf, T, c.lo, c.hi, w, g);
        T += 128;
    }

    // the waves' columns, [wave][column][D + 4], and their references and sums (-1: nothing seen)
    constexpr uint32_t PITCH = D + 4;
    float *sm = lds + 64 * PITCH, *sl = sm + 64;
    const float l = column_sum4(st.l);
    const bool seen = column_max4(st.seen ? 1.0f : 0.0f) > 0.0f;
    if (n < cols) {
        float *to = lds + (wave * cols + n) * PITCH;
        const float f = st.vref * 0.0078125f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 16; j += 4)
                *(f32x4 *)(to + (4 * g + i) * (D / 16) + j) =
                    f32x4{st.o[j][i] * f, st.o[j + 1][i] * f, st.o[j + 2][i] * f, st.o[j + 3][i] * f};
        if (g == 0) {
            sm[wave * 16 + n] = st.m;
            sl[wave * 16 + n] = seen ? l : -1.0f;
        }
    }
    __syncthreads();
    for (uint32_t at = tid; at < cols * (D / 4); at += ER_KV8_THREADS) {
        const uint32_t col = at / (D / 4), d = (at % (D / 4)) * 4;
        float m = ER_NO_MAX, total = 0.0f;
        bool visible = false;
#pragma unroll
        for (int v = 0; v < 4; ++v) m = fmaxf(m, sm[v * 16 + col]);
        f32x4 o = {};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float part = sl[v * 16 + col];
            if (part < 0.0f) continue;
            visible = true;
            const float f = __builtin_amdgcn_exp2f(sm[v * 16 + col] - m);
            total += part * f;
            o += *(const f32x4 *)(lds + (v * cols + col) * PITCH + d) * f;
        }
        const Column k = column_of(p, q, h, col);
        if (p.splits == 1) {
            const float r = quotient(total, visible);
            store4(p, k.row, k.head, d, D, visible ? o * r : f32x4{});
        } else {
            const size_t to = part_index(p, piece, k.row, k.head);
            if (visible) *(f32x4 *)(p.partO + to * D + d) = o;
            if (d == 0) {
                p.partML[2 * to] = m;
                p.partML[2 * to + 1] = visible ? total : -1.0f;
            }
        }
    }
}

// ---------------------------------------------------------------- many columns: prefill

#define ER_WIDE_TOKENS 64

// What a tile's four 16-token parts bring: page, scales.
struct WideParts {
    int page[4];
    float ks[4], vs[4];
};
template <int D>
struct WideTile {
    u32x4 k[D / 64];                       // token tid / 4, bytes [(tid & 3) D/4, + D/4)
    uint32_t v[(D + 127) / 128][8];        // see value_item
};

ER_DEV void wide_pages(WideParts &w, const ErAttendArgs &p, uint32_t s, int T, int lo, int hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = T + 16 * i;
        w.page[i] = at < hi && at + 16 > lo ? uniform(page_of(p.b, p.c, s, at)) : -1;
    }
}
ER_DEV void wide_scales(WideParts &w, const ErAttendArgs &p, uint32_t h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const size_t block = (size_t)(uint32_t)max(w.page[i], 0) * p.c.heads + h;
        w.ks[i] = p.c.ks[block];
        w.vs[i] = p.c.vs[block];
    }
}
// v[i] for an index that differs between lanes, without an address (which would put v into scratch memory)
template <typename T>
ER_DEV T pick4(const T (&v)[4], uint32_t i) {
    const T a = v[0], b = v[1], c = v[2], d = v[3];
    const T x = i & 1u ? b : a, y = i & 1u ? d : c;
    return i & 2u ? y : x;
}

// Item `it` of a tile's values: four codes (dword) of the eight tokens (first
// .. first + 3, first + 8 .. first + 11) that one lane half holds of a
// 16-token slice of S^T.
struct ValueItem {
    uint32_t slot, dword, part;
    int first;
};
template <int D>
ER_DEV ValueItem value_item(uint32_t it) {
    ValueItem v;
    v.slot = it / (D / 4);
    v.dword = it % (D / 4);
    v.part = v.slot >> 1;
    v.first = (int)(16 * v.part + 4 * (v.slot & 1));
    return v;
}

template <int D>
ER_DEV void load_wide(WideTile<D> &t, const WideParts &w, const ErAttendArgs &p, uint32_t h, int T, uint32_t tid) {
    const uint32_t mask = (1u << p.c.shift) - 1u;
    {
        const uint32_t tok = tid >> 2;
        const size_t block = (size_t)(uint32_t)max(pick4(w.page, tok >> 4), 0) * p.c.heads + h;
        const uint8_t *src = p.c.k + ((block << p.c.shift) + (((uint32_t)T + tok) & mask)) * D + (tid & 3u) * (D / 4);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) t.k[j] = *(const u32x4 *)(src + 16 * j);
    }
#pragma unroll
    for (int r = 0; r < (D + 127) / 128; ++r) {
        const ValueItem it = value_item<D>((tid + 256 * r) & (2 * D - 1));  // D = 64: half the threads repeat
        const size_t block = (size_t)(uint32_t)max(pick4(w.page, it.part), 0) * p.c.heads + h;
        const uint8_t *src = p.c.v + ((block << p.c.shift) + (((uint32_t)T + (uint32_t)it.first) & mask)) * D + 4 * it.dword;
#pragma unroll
        for (int i = 0; i < 8; ++i) t.v[r][i] = *(const uint32_t *)(src + ((i & 3) + 8 * (i >> 2)) * D);
    }
}

// LDS: keys [64][D + 8], values transposed [D][64 + 8], both fp16; a flag a
// wave for NaN codes.  The pitches put consecutive rows 4 banks apart.
template <int D>
struct WideLds {
    _Float16 k[ER_WIDE_TOKENS][D + 8];
    _Float16 v[D][ER_WIDE_TOKENS + 8];
};

template <int D>
ER_DEV bool store_wide(WideLds<D> &to, const WideTile<D> &t, const WideParts &w, float vref, int T, int lo, int hi,
                       uint32_t tid) {
    {
        _Float16 *dst = &to.k[tid >> 2][(tid & 3u) * (D / 4)];
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            *(h8 *)(dst + 16 * j) = codes_to_h8(t.k[j].x, t.k[j].y);
            *(h8 *)(dst + 16 * j + 8) = codes_to_h8(t.k[j].z, t.k[j].w);
        }
    }
    bool nan = false;
#pragma unroll
    for (int r = 0; r < (D + 127) / 128; ++r) {
        const ValueItem it = value_item<D>((tid + 256 * r) & (2 * D - 1));
        const bool ok = pick4(w.page, it.part) >= 0;
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // tokens that no column sees, or without a page, count as zeros whatever their bytes hold
            const int tok = T + it.first + (i & 3) + 8 * (i >> 2);
            c[i] = ok && tok >= lo && tok < hi ? t.v[r][i] : 0u;
            nan |= (((c[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }
        h8 a[4];
        const float f = ok ? 128.0f * (pick4(w.vs, it.part) / vref) : 1.0f;
        transpose_codes(c, f, f, a);
#pragma unroll
        for (int j = 0; j < 4; ++j) *(h8 *)&to.v[4 * it.dword + j][8 * it.slot] = a[j];
    }
    return nan;
}

ER_DEV float column_max2(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
ER_DEV float column_sum2(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <int TERMS>
ER_DEV void add_values32(f32x16 &o, h8 a, const h8 (&b)[TERMS], h8 visible, bool nans) {
    if (!nans) {
#pragma unroll
        for (int term = 0; term < TERMS; ++term) o = mfma32(a, b[term], o);
        return;
    }
    const f32x16 hits = mfma32(nan_places(a), visible, f32x16{});
    a = without_nan(a);
#pragma unroll
    for (int term = 0; term < TERMS; ++term) o = mfma32(a, b[term], o);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = hits[i] > 0.0f ? __builtin_nanf("") : o[i];
}

// 128 columns against one piece of their sequence's tokens, 32 columns a wave:
// bound by the matrix products and the softmax's exponentials.  The four waves
// convert each 64-token tile to fp16 once, into LDS, while the tile before is
// worked on; a lane half's tokens of a slice lie together there, so that one
// 16-byte read is an operand.
template <int D, int TERMS>
ER_DEV void kv8_attend_wide(const ErAttendArgs &p, WideLds<D> *lds, uint32_t (*nanFlags)[4]) {
    // units (sequence, head, piece) are dealt over a multiple of 8 workgroups,
    // and workgroups to the 8 XCDs in turn, so that one XCD's L2 serves all
    // row tiles of a unit; later row tiles see more tokens and start first
    const uint32_t units = p.b.sequences * p.c.heads * p.splits, dealt = (units + 7u) & ~7u;
    const uint32_t unit = blockIdx.x % dealt, tile = p.tiles - 1 - blockIdx.x / dealt;
    if (unit >= units) return;
    const uint32_t piece = unit % p.splits, h = (unit / p.splits) % p.c.heads, s = unit / p.splits / p.c.heads;
    const Sequence q = sequence_of(p.b, s);
    const uint32_t cols = (uint32_t)q.n * p.group, col0 = tile * 128;
    if (col0 >= cols) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), n = lane & 31u, hh = lane >> 5;
    const Spans w = spans_of(p, q, col0, min(col0 + 127, cols - 1));
    const uint32_t wcol0 = col0 + 32 * wave;
    const bool idle = wcol0 >= cols;  // this wave has no columns; it converts all the same
    const Spans ww = spans_of(p, q, min(wcol0, cols - 1), min(wcol0 + 31, cols - 1));
    const Column c = column_of(p, q, h, min(wcol0 + n, cols - 1));
    const bool live = wcol0 + n < cols;
    const int begin = (w.anyLo & ~63) + (int)(piece * p.chunk), end = min(w.anyHi, begin + (int)p.chunk);

    f32x16 o[D / 32] = {};
    float m = ER_NO_MAX, l = 0.0f, vref = 0.0f;
    bool seen = false;
    if (begin < end) {
        WideTile<D> t;
        WideParts now, next;
        wide_pages(now, p, s, begin, w.anyLo, end);
        wide_pages(next, p, s, begin + 64, w.anyLo, end);
        load_wide<D>(t, now, p, h, begin, tid);
        wide_scales(now, p, h);
        h8 qb[TERMS][D / 16];
        const float qf = load_query<D / 16, TERMS>(p.q + (size_t)c.row * p.qStride + (size_t)c.head * D, live, hh * 8, 16,
                                                   qb, column_max2) * p.scale;
        float shrink = 0.0f;
        auto raise = [&](const WideParts &parts) {  // the value scales' reference, and what it does to o
            float top = vref;
#pragma unroll
            for (int i = 0; i < 4; ++i) top = parts.page[i] >= 0 ? fmaxf(top, parts.vs[i]) : top;
            shrink = top > vref ? vref / top : 1.0f;
            vref = top;
        };
        raise(now);
        bool nan = store_wide<D>(lds[0], t, now, vref, begin, w.anyLo, end, tid);
        nan = __any(nan);
        if (lane == 0) nanFlags[0][wave] = nan;
        uint32_t buf = 0;
        for (int T = begin; T < end; T += 64, buf ^= 1u) {
            __syncthreads();
            const WideParts parts = now;
            const float rescale = shrink;
            const bool more = T + 64 < end;
            if (more) {
                now = next;
                load_wide<D>(t, now, p, h, T + 64, tid);
                wide_scales(now, p, h);
                wide_pages(next, p, s, T + 128, w.anyLo, end);
            }
            bool none = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) none &= parts.page[i] < 0;
            if (rescale != 1.0f) {
#pragma unroll
                for (int d = 0; d < D / 32; ++d) o[d] *= rescale;
            }
            if (!idle && !none && T < ww.anyHi && T + 64 > ww.anyLo) {
                const WideLds<D> &in = lds[buf];
                float x[2][16];
#pragma unroll
                for (int th = 0; th < 2; ++th) {
                    f32x16 sc = {};
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const h8 a = *(const h8 *)&in.k[32 * th + n][16 * k + 8 * hh];
#pragma unroll
                        for (int term = 0; term < TERMS; ++term) sc = mfma32(a, qb[term][k], sc);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[th][i] = sc[i] * (qf * parts.ks[2 * th + (i >> 3)]);
                }
                bool whole = T >= ww.allLo && T + 64 <= ww.allHi;
#pragma unroll
                for (int i = 0; i < 4; ++i) whole &= parts.page[i] >= 0;
                uint32_t shown = ~0u;
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int tok = T + 32 * (i >> 4) + 8 * ((i & 15) >> 2) + 4 * (int)hh + (i & 3);
                        if (!(parts.page[i >> 3] >= 0 && tok >= c.lo && tok < c.hi)) {
                            x[i >> 4][i & 15] = -__builtin_inff();
                            shown &= ~(1u << i);
                        }
                    }
                }
                seen |= shown != 0;
                float top = x[0][0];
#pragma unroll
                for (int i = 1; i < 32; ++i) top = fmaxf(top, x[i >> 4][i & 15]);
                if (__any(top > m + 8.0f)) {
                    const float mm = fmaxf(m, column_max2(top));
                    const float f = __builtin_amdgcn_exp2f(m - mm);
                    m = mm;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d) o[d] *= f;
                }
                const bool nans = !whole && (nanFlags[buf][0] | nanFlags[buf][1] | nanFlags[buf][2] | nanFlags[buf][3]);
#pragma unroll
                for (int sl = 0; sl < 4; ++sl) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        e[i] = __builtin_amdgcn_exp2f(x[sl >> 1][8 * (sl & 1) + i] - (m - 7.0f));
                        l += e[i];
                    }
                    h8 b[TERMS], visible;
                    weight_terms<TERMS>(e, b);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        visible[i] = (shown >> (8 * sl + i)) & 1u ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
                        add_values32<TERMS>(o[d], *(const h8 *)&in.v[32 * d + n][16 * sl + 8 * hh], b, visible, nans);
                }
            }
            if (more) {
                raise(now);
                bool nn = store_wide<D>(lds[buf ^ 1u], t, now, vref, T + 64, w.anyLo, end, tid);
                nn = __any(nn);
                if (lane == 0) nanFlags[buf ^ 1u][wave] = nn;
            }
        }
    }
    l = column_sum2(l);
    seen = column_max2(seen ? 1.0f : 0.0f) > 0.0f;
    if (!live) return;
    const float unitOf = vref * 0.0078125f;
    const float f = p.splits == 1 ? (seen ? unitOf / l : 0.0f) : unitOf;
    const size_t to = part_index(p, piece, c.row, c.head);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at = 32 * d + 8 * i + 4 * hh;
            f32x4 v = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * f;
            if (p.splits == 1)
                store4(p, c.row, c.head, at, D, seen ? v : f32x4{});
            else if (seen)
                *(f32x4 *)(p.partO + to * D + at) = v;
        }
    if (p.splits > 1 && hh == 0) {
        p.partML[2 * to] = m;
        p.partML[2 * to + 1] = seen ? l : -1.0f;
    }
}

// ---------------------------------------------------------------- joining the pieces

// One row and head's pieces: weights 2^(m - max) / sum from the references and
// sums, then the weighted outputs; a quarter of the pieces to each wave.
template <int D>
ER_DEV void kv8_join(const ErAttendArgs &p, float *lds) {
    const uint32_t heads = p.group * p.c.heads, row = blockIdx.x / heads, head = blockIdx.x % heads;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6);
    const uint32_t s = uniform(sequence_of_row(p.b, row, lane));
    if (s >= p.b.sequences) return;
    const Sequence q = sequence_of(p.b, s);
    if ((int)row < q.row0 || (int)row >= q.row0 + q.n) return;
    float *weight = lds, *red = lds + ((p.splits + 3u) & ~3u);  // [splits], [4][D]
    float top = ER_NO_MAX;
    for (uint32_t i = lane; i < p.splits; i += 64) top = fmaxf(top, p.partML[2 * part_index(p, i, (int)row, head)]);
#pragma unroll
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    float total = 0.0f;
    bool seen = false;
    for (uint32_t i = lane; i < p.splits; i += 64) {
        const size_t at = 2 * part_index(p, i, (int)row, head);
        const float l = p.partML[at + 1];
        const float f = l < 0.0f ? -1.0f : __builtin_amdgcn_exp2f(p.partML[at] - top);
        if (!(l < 0.0f)) {
            total += l * f;
            seen = true;
        }
        if (wave == 0) weight[i] = f;
    }
    // every wave has the sum, of the same terms in the same order
#pragma unroll
    for (int x = 32; x; x >>= 1) total += __shfl_xor(total, x);
    seen = __any(seen);
    __syncthreads();
    constexpr int PER = D / 64;
    float o[PER] = {};
    for (uint32_t i = wave; i < p.splits; i += 4) {
        const float f = weight[i];
        if (f < 0.0f) continue;
        const float *src = p.partO + part_index(p, i, (int)row, head) * D + lane * PER;
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] += f * src[j];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) red[wave * D + lane * PER + j] = o[j];
    __syncthreads();
    if (tid < D / 4) {
        f32x4 v = {};
#pragma unroll
        for (int k = 0; k < 4; ++k) v += *(const f32x4 *)(red + k * D + 4 * tid);
        store4(p, (int)row, head, 4 * tid, D, seen ? v * quotient(total, true) : f32x4{});
    }
}

extern __shared__ __attribute__((aligned(16))) float er_kv8_lds[];

#define ER_KV8_ATTEND(D, TERMS, NAME, NARROW, WAVES)                                                               \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS, NARROW)                                           \
        er_kv8_attend_narrow_d##D##_##NAME(ErAttendArgs p) {                                                       \
        __shared__ __attribute__((aligned(16))) float sums[64 * (D + 4) + 128];                                    \
        kv8_attend_narrow<D, TERMS>(p, sums);                                                                      \
    }                                                                                                              \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS, WAVES)                                            \
        er_kv8_attend_wide_d##D##_##NAME(ErAttendArgs p) {                                                         \
        __shared__ WideLds<D> tiles[2];                                                                            \
        __shared__ uint32_t nanFlags[2][4];                                                                        \
        kv8_attend_wide<D, TERMS>(p, tiles, nanFlags);                                                             \
    }
ER_KV8_ATTEND(64, 1, bf16, 2, 2)
ER_KV8_ATTEND(64, 2, f32, 2, 2)
ER_KV8_ATTEND(128, 1, bf16, 2, 2)
ER_KV8_ATTEND(128, 2, f32, 2, 1)
ER_KV8_ATTEND(256, 1, bf16, 1, 1)
ER_KV8_ATTEND(256, 2, f32, 1, 1)

#define ER_KV8_JOIN(D)                                                                                             \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS) er_kv8_join_d##D(ErAttendArgs p) {                \
        kv8_join<D>(p, er_kv8_lds);                                                                                \
    }
ER_KV8_JOIN(64)
ER_KV8_JOIN(128)
ER_KV8_JOIN(256)
