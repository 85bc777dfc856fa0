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
// by more than 2 (in powers of two); weights are 2^(s - m + 13), so at most
// 2^15, and the reference cancels in the quotient.  Most tiles rescale nothing.
// fp16's smallest step, 2^-24, is then 2^-37 of the row's largest weight at the
// most: what the rounding of smaller weights leaves out of 2^18 tokens is 2^-20
// of their values.  By 8 and + 7, which rescales less, it was 2^-14; a prompt of
// 4096 rows then took 183.4 us where it takes 185.3 so.

#define ER_SLACK 2.0f
#define ER_LIFT 13.0f
#define ER_NO_MAX (-3.0e38f)  // reference of a column that has seen no score

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

// A byte of ones for each NaN code of a dword.
ER_DEV uint32_t nan_codes(uint32_t c) {
    const uint32_t top = ((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // 0x7f alone carries into bit 7
    return (top << 1) - (top >> 7);
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

// A column's query times the softmax's scale (and log2 e) as B operands: eight
// consecutive values for each of N products, those of product k from `from` +
// k / 2 * pair + k % 2 * next on, as one or two fp16 terms.  It is brought to below 1 by a power of two
// over the whole head (`join_lanes` takes the largest magnitude over the lanes
// that share the column); returns that power.  With the keys' scales powers of
// two as well, a score is its product times a power of two, exactly: the fused
// multiply-add that takes the reference off it and the product that the
// reference was taken from agree to the last bit, however large the scores.
template <int N, int TERMS, typename JOIN>
ER_DEV float load_query(const float *src, bool live, float scale, uint32_t from, uint32_t pair, uint32_t next,
                        h8 (&b)[TERMS][N], JOIN join_lanes) {
    float x[N][8];
    float peak = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        f32x4 lo = {}, hi = {};
        if (live) {
            const float *v = src + from + k / 2 * pair + k % 2 * next;
            lo = *(const f32x4_a4 *)v;
            hi = *(const f32x4_a4 *)(v + 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[k][i] = lo[i] * scale;
            x[k][4 + i] = hi[i] * scale;
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

// The factor of a 16-token part's scores.  Not 0, so that -inf stays the score
// of a hidden token.
ER_DEV float score_factor(float qf, float ks) { return fmaxf(qf * ks, 1.2e-38f); }

// Weights of eight tokens as one or two fp16 terms.  The pair is hidden from
// the compiler (by no instruction at all), which else converts a first term
// twice, packed for the product and single for the second term.
ER_DEV h2 to_h2(float a, float b) {
    h2 r = {(_Float16)a, (_Float16)b};
    asm("" : "+v"(r));
    return r;
}
template <int TERMS>
ER_DEV void weight_terms(const float w[8], h8 (&b)[TERMS]) {
    const h2 p0 = to_h2(w[0], w[1]), p1 = to_h2(w[2], w[3]), p2 = to_h2(w[4], w[5]), p3 = to_h2(w[6], w[7]);
    b[0] = join(p0, p1, p2, p3);
    if constexpr (TERMS == 2) {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = __builtin_fmaf((float)b[0][i], -1.0f, w[i]);
        b[1] = join(to_h2(r[0], r[1]), to_h2(r[2], r[3]), to_h2(r[4], r[5]), to_h2(r[6], r[7]));
    }
}

typedef __bf16 b16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
ER_DEV void store4(const ErAttendArgs &p, int row, uint32_t head, uint32_t d, uint32_t D, f32x4 v) {
    const size_t at = (size_t)row * p.outStride + (size_t)head * D + d;
    if (p.half)
        *(b16x4_a2 *)((uint16_t *)p.out + at) = b16x4_a2{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
    else
        *(f32x4_a4 *)((float *)p.out + at) = v;
}
// Index of a column's partial sums of one piece.
ER_DEV size_t part_index(const ErAttendArgs &p, uint32_t piece, int row, uint32_t head) {
    return ((size_t)piece * p.b.rows + (size_t)row) * (p.group * p.c.heads) + head;
}
// A column's output is its sums over l; zeros where no token is visible.
// Where some are and l is 0 or NaN (scores without a finite maximum), the
// quotient is NaN, as the softmax's is.  Sums that are joined are divided by
// their own l first and weighted by its share of the whole, so that a mean of
// values near fp32's largest stays inside its range.
ER_DEV float over(float l) { return l != 0.0f ? 1.0f / l : 1.0f; }
ER_DEV float share_of(float l, float total) { return total != 0.0f ? l / total : 0.0f; }
ER_DEV f32x4 joined(f32x4 o, bool visible, float total) {
    return !visible ? f32x4{} : total != 0.0f ? o : o + __builtin_nanf("");
}

// ---------------------------------------------------------------- few columns: decode, drafts

// One 32-token tile of keys and values in registers, as loaded.
template <int D>
struct NarrowTile {
    u32x4 k[2][D / 64];      // lane (n, g): token n of each half, bytes 64 j + 16 g .. + 15 (a load reads 64 bytes of a row)
    uint32_t v[D / 64][8];   // lane (n, g): tokens 4 g + i of the first half, then of the second, bytes [n D/16, (n + 1) D/16)
    float ks[2], vs[2];      // the halves' scales
    int page[2];             // the halves' pages; -1: outside the pool, or no visible token
};

// The pages of a tile's halves, found a tile ahead of its loads.
struct NarrowPages {
    int page[2];
};
template <int P>
ER_DEV NarrowPages narrow_pages(const ErAttendArgs &p, uint32_t s, int T, int lo, int hi) {
    NarrowPages w;
    constexpr int AT = P < 32 ? 16 : 32;  // tokens that one entry covers
    auto page = [&](int at) { return at < hi && at + AT > lo ? uniform(page_of(p.b, p.c, s, at)) : -1; };
    w.page[0] = page(T);
    w.page[1] = P < 32 ? page(T + 16) : w.page[0];
    return w;
}

template <int D, int P>
ER_DEV void load_narrow(NarrowTile<D> &t, const NarrowPages &w, const ErAttendArgs &p, uint32_t h, int T, uint32_t n,
                        uint32_t g) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        t.page[half] = w.page[half];
        const size_t block = (size_t)(uint32_t)max(w.page[half], 0) * p.c.heads + h;
        if (half == 0 || P < 32) {
            t.ks[half] = load_shared(p.c.ks + block);
            t.vs[half] = load_shared(p.c.vs + block);
        } else {
            t.ks[1] = t.ks[0];
            t.vs[1] = t.vs[0];
        }
        const size_t base = block * (P * D) + ((uint32_t)(T + 16 * half) % P) * D;
        const uint8_t *kp = p.c.k + base + (n * D + 16 * g);
        const uint8_t *vp = p.c.v + base + (4 * g * D + n * (D / 16));
#pragma unroll
        for (int j = 0; j < D / 64; ++j) t.k[half][j] = *(const u32x4 *)(kp + 64 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (D == 64) {
                t.v[0][4 * half + i] = *(const uint32_t *)(vp + i * D);
            } else if constexpr (D == 128) {
                const u32x2 x = *(const u32x2 *)(vp + i * D);
                t.v[0][4 * half + i] = x.x;
                t.v[1][4 * half + i] = x.y;
            } else {
                const u32x4 x = *(const u32x4 *)(vp + i * D);
                t.v[0][4 * half + i] = x.x;
                t.v[1][4 * half + i] = x.y;
                t.v[2][4 * half + i] = x.z;
                t.v[3][4 * half + i] = x.w;
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
    float vref, vinv; // reference of the value scales: o is in units of vref / 128; 128 / vref (wave-uniform)
    bool seen;        // a token was visible to the column
    bool nans;        // a masked tile held NaN codes
};

// Tokens that some column sees, and tokens that every column sees.
struct Spans {
    int anyLo, anyHi, allLo, allHi;
};
ER_DEV Spans spans_of(const ErAttendArgs &p, const Sequence &q, uint32_t firstCol, uint32_t lastCol) {
    const Column a = column_of(p, q, 0, firstCol), b = column_of(p, q, 0, lastCol);
    return Spans{a.lo, b.hi, b.lo, a.hi};
}

// Moves a column's reference up to its scores' largest.
template <int N, typename ACC>
ER_DEV void raise_reference(float to, float &m, float &l, ACC (&o)[N]) {
    const float f = __builtin_amdgcn_exp2f(m - to);
    m = to;
    l *= f;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= f;
}
// Moves the value scales' reference.
template <int N, typename ACC>
ER_DEV void raise_scale(float to, float &vref, float &vinv, ACC (&o)[N]) {
    const float f = vref / to;
    vref = to;
    vinv = 128.0f / to;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= f;
}

// Value scales as integers, which order as the (positive) floats do.  More than
// 2^22 below the reference, a part's smallest codes fall below fp16's.
#define ER_SCALE_APART (22u << 23)
struct ScaleRange {
    uint32_t most, least;  // of the parts that are there; least: of those that are not 0, less one
    __device__ __forceinline__ void add(uint32_t scale) {
        most = max(most, scale);
        least = min(least, scale - 1u);
    }
    __device__ __forceinline__ bool apart() const { return most > least && most - least > ER_SCALE_APART; }
};
// Moves the reference of the value scales for the parts at hand: up to the
// largest; and down to it where one lies too far below, since the reference may
// stem from tokens that only others of the wave's columns see.  Sums, at most
// 2^61, are rescaled exactly: by at most 2^60 below the largest reference, `top`.
template <int N, typename ACC>
ER_DEV void follow_scale(const ScaleRange &r, float &top, float &vref, float &vinv, ACC (&o)[N]) {
    const uint32_t ref = __float_as_uint(vref);
    const bool up = r.most > ref, down = r.most < ref && ref > ER_SCALE_APART && r.least < ref - ER_SCALE_APART;
    if (!up && !down) return;
    const float to = fmaxf(__uint_as_float(r.most), top * 0x1p-60f);
    top = fmaxf(top, to);
    raise_scale(to, vref, vinv, o);
}

// One tile into the state.  MASKED: some column does not see all of it, or a
// page is missing.  Hidden tokens get the score -inf there, and those that no
// column sees have their bytes taken as zeros, whatever they hold.  NaN codes
// count as zeros too, since a column may not see them and 0 * NaN is NaN:
// st.nans remembers that there were some, and mark_nans brings them back.
// vtop: the largest reference of the value scales, for masked tiles, which come
// last.
template <int D, int TERMS, bool MASKED>
ER_DEV void attend_narrow(NarrowState<D> &st, NarrowTile<D> &t, const h8 (&qb)[TERMS][D / 32], float qf, int T,
                          int lo, int hi, const Spans &w, uint32_t g, float &vtop) {
    const bool ok0 = !MASKED || t.page[0] >= 0, ok1 = !MASKED || t.page[1] >= 0;
    f32x4 s[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        s[half] = f32x4{};
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const u32x4 c = t.k[half][k / 2];
            const h8 a = k % 2 ? codes_to_h8(c.z, c.w) : codes_to_h8(c.x, c.y);
#pragma unroll
            for (int term = 0; term < TERMS; ++term) s[half] = mfma16(a, qb[term][k], s[half]);
        }
    }
    if constexpr (!MASKED) {
        st.seen = true;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int tok = T + 16 * (i / 4) + 4 * (int)g + (i & 3);
            const bool ok = i < 4 ? ok0 : ok1, shown = ok && tok >= lo && tok < hi;
            st.seen |= shown;
            s[i / 4][i & 3] = shown ? s[i / 4][i & 3] : -__builtin_inff();
#pragma unroll
            for (int d = 0; d < D / 64; ++d) {
                const uint32_t c = ok && tok >= w.anyLo && tok < w.anyHi ? t.v[d][i] : 0u, nan = nan_codes(c);
                st.nans |= nan != 0;
                t.v[d][i] = c & ~nan;
            }
        }
    }
    const float f0 = score_factor(qf, ok0 ? t.ks[0] : t.ks[1]), f1 = score_factor(qf, ok1 ? t.ks[1] : t.ks[0]);
    const float top = fmaxf(fmaxf(fmaxf(s[0].x, s[0].y), fmaxf(s[0].z, s[0].w)) * f0,
                            fmaxf(fmaxf(s[1].x, s[1].y), fmaxf(s[1].z, s[1].w)) * f1);
    if (__any(top > st.m + ER_SLACK)) raise_reference(fmaxf(st.m, column_max4(top)), st.m, st.l, st.o);
    const float vs0 = ok0 ? t.vs[0] : t.vs[1], vs1 = ok1 ? t.vs[1] : t.vs[0];
    if constexpr (MASKED) {
        ScaleRange r = {0u, ~0u};
        r.add(__float_as_uint(uniform(vs0)));
        r.add(__float_as_uint(uniform(vs1)));
        follow_scale(r, vtop, st.vref, st.vinv, st.o);
    } else if (fmaxf(vs0, vs1) > st.vref) {
        raise_scale(fmaxf(vs0, vs1), st.vref, st.vinv, st.o);
    }
    const float v0 = vs0 * st.vinv, v1 = vs1 * st.vinv, base = st.m - ER_LIFT;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(s[i / 4][i & 3] * (i < 4 ? f0 : f1) - base);
    st.l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    h8 b[TERMS];
    weight_terms<TERMS>(x, b);
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
        h8 a[4];
        transpose_codes(t.v[d], v0, v1, a);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int term = 0; term < TERMS; ++term) st.o[4 * d + j] = mfma16(a[j], b[term], st.o[4 * d + j]);
    }
}

// The sums that a visible NaN code of the masked tiles belongs to become NaN.
// Reached only where such a tile held one, so it takes the tokens one by one.
template <int D>
ER_DEV void mark_nans(NarrowState<D> &st, const ErAttendArgs &p, uint32_t s, uint32_t h, int begin, int end, int lo,
                      int hi, uint32_t g) {
    for (int tok = max(begin, lo); tok < min(end, hi); ++tok) {
        const int page = page_of(p.b, p.c, s, tok);
        if (page < 0) continue;
        const size_t slot = (((size_t)page * p.c.heads + h) << p.c.shift) + ((uint32_t)tok & ((1u << p.c.shift) - 1u));
        const uint8_t *v = p.c.v + slot * D;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < D / 64; ++d) {
                const uint32_t nan = nan_codes(*(const uint32_t *)(v + (4 * g + i) * (D / 16) + 4 * d));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    st.o[4 * d + j][i] = (nan >> (8 * j)) & 1u ? __builtin_nanf("") : st.o[4 * d + j][i];
            }
    }
}

template <int N>
struct Const {
    static constexpr int value = N;
};

// How the tokens of all sequences and heads are shared between workgroups.
// Units (sequence, head, block of 16 columns) lie one behind the other, each `length` steps of 64
// tokens long, and workgroup w takes steps w * quota .. (w + 1) * quota - 1 of
// that line: whatever the sequences' lengths, all have the same to read, and a
// workgroup's start (some microseconds of dependent loads) is paid once for each
// that is resident.  Pieces of one length took 150 us for 64 ragged users where
// this takes 123, four times as many 162.  Where there is so little that each takes the least, units begin at multiples
// of it, so that no workgroup takes two.
struct Shares {
    uint32_t quota, total;
    bool aligned;
};
ER_DEV uint32_t steps_of(const ErAttendArgs &p, const Sequence &q) {
    if (q.n == 0) return 0;
    const Spans w = spans_of(p, q, 0, (uint32_t)q.n * p.group - 1);
    // rows that see nothing take a step all the same, which writes their zeros
    return max(1u, ((uint32_t)max(w.anyHi - (w.anyLo & ~63), 0) + 63u) >> 6);
}
// Column blocks of a sequence and key/value head.
ER_DEV uint32_t blocks_of(const ErAttendArgs &p, const Sequence &q) { return ((uint32_t)q.n * p.group + 15u) >> 4; }
ER_DEV uint32_t shared_length(const ErAttendArgs &p, uint32_t steps, bool aligned) {
    return aligned ? (steps + p.least - 1) / p.least * p.least : steps;
}
// Inclusive prefix sum over the wave: within rows of 16 lanes, then row ends
// into the rows behind.
ER_DEV uint32_t wave_prefix(uint32_t v) {
    auto from = [](uint32_t x, auto ctrl, auto rows) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    v += from(v, Const<0x111>{}, Const<0xf>{});  // lanes 1, 2, 4 and 8 before
    v += from(v, Const<0x112>{}, Const<0xf>{});
    v += from(v, Const<0x114>{}, Const<0xf>{});
    v += from(v, Const<0x118>{}, Const<0xf>{});
    v += from(v, Const<ER_DPP_ROW_BCAST15>{}, Const<0xa>{});
    v += from(v, Const<ER_DPP_ROW_BCAST31>{}, Const<0xc>{});
    return v;
}
ER_DEV uint32_t lane_of(uint32_t v, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane); }
ER_DEV uint32_t wave_sum(uint32_t v) { return lane_of(wave_prefix(v), 63); }

// Lane i's sequence of the first 64, loaded once: most batches have no more,
// and what a workgroup needs to know of others then passes between lanes.
struct LaneSequence {
    Sequence q;
    uint32_t steps;
};
ER_DEV LaneSequence lane_sequence(const ErAttendArgs &p, uint32_t s) {
    LaneSequence l = {};
    if (s < p.b.sequences) {
        l.q = sequence_of(p.b, s);
        l.steps = steps_of(p, l.q);
    }
    return l;
}
ER_DEV LaneSequence lane_sequence_at(const ErAttendArgs &p, const LaneSequence &first, uint32_t s) {
    if (s >= 64) return lane_sequence(p, s);
    LaneSequence l;
    l.q.row0 = (int)lane_of((uint32_t)first.q.row0, s);
    l.q.n = (int)lane_of((uint32_t)first.q.n, s);
    l.q.len = (int)lane_of((uint32_t)first.q.len, s);
    l.steps = lane_of(first.steps, s);
    return l;
}
ER_DEV Shares shares_of(const ErAttendArgs &p, const LaneSequence &first, uint32_t lane) {
    uint32_t plain = first.steps * blocks_of(p, first.q), padded = shared_length(p, first.steps, true) * blocks_of(p, first.q);
    for (uint32_t at = 64; at < p.b.sequences; at += 64) {
        const LaneSequence l = lane_sequence(p, at + lane);
        plain += l.steps * blocks_of(p, l.q);
        padded += shared_length(p, l.steps, true) * blocks_of(p, l.q);
    }
    plain = wave_sum(plain) * p.c.heads;
    padded = wave_sum(padded) * p.c.heads;
    Shares s;
    s.aligned = padded <= p.shares * p.least;
    s.total = s.aligned ? padded : plain;
    s.quota = s.aligned ? p.least : max(p.least, (plain + p.shares - 1) / p.shares);
    return s;
}
// The sequence that step `at` of the line belongs to, and where it begins.
ER_DEV uint32_t sequence_at(const ErAttendArgs &p, const LaneSequence &first, bool aligned, uint32_t at, uint32_t lane,
                            uint32_t &begins) {
    uint32_t before = 0;
    for (uint32_t s0 = 0;; s0 += 64) {
        const LaneSequence l = s0 ? lane_sequence(p, s0 + lane) : first;
        const uint32_t mine = shared_length(p, l.steps, aligned) * blocks_of(p, l.q) * p.c.heads, upTo = wave_prefix(mine);
        const uint64_t past = __ballot(before + upTo > at);
        if (past || s0 + 64 >= p.b.sequences) {
            const uint32_t i = past ? (uint32_t)__ffsll((unsigned long long)past) - 1u : 63u;
            begins = before + lane_of(upTo - mine, i);
            return s0 + i;
        }
        before += lane_of(upTo, 63);
    }
}

// Up to 16 columns from col0 on (rows of one sequence times query heads of one
// key/value head) against steps [from, to) of their tokens: bound by the bytes of the
// cache.  Every wave takes each fourth 32-token tile straight into registers,
// 8 KB of codes at head width 128, with the next tile in flight while it
// works; keys and values need no exchange between lanes, so nothing passes
// through LDS until the waves' sums are joined at the end.  The sums of all
// steps are the columns' outputs; else they go to part `part`.  64 ragged users
// of an 8B layer (675 MB of codes) take 123 us, 131072 tokens of one user (268
// MB) 50 us: 5.4 to 5.5 TB/s, a large read's rate.
template <int D, int P, int TERMS>
ER_DEV void narrow_unit(const ErAttendArgs &p, uint32_t s, const Sequence &q, uint32_t h, uint32_t col0, uint32_t from,
                        uint32_t to, bool complete, uint32_t part, float *lds) {
    // what follows from the thread's index is formed for each unit: kept from one to the next, it takes registers
    // that head width 256 needs for its tile
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const uint32_t lane = tid & 63u, wave = uniform(tid >> 6), n = lane & 15u, g = lane >> 4;
    const uint32_t every = (uint32_t)q.n * p.group, cols = min(every - col0, 16u);
    const Spans w = spans_of(p, q, col0, col0 + cols - 1);
    const int base = column_of(p, q, h, 0).lo & ~63;  // the steps are those of all columns
    const int begin = base + 64 * (int)from, end = min(w.anyHi, base + 64 * (int)to);
    const Column c = column_of(p, q, h, col0 + min(n, cols - 1));

    // The tiles that all columns see whole go through a loop of their own, two
    // in registers at a time; the few others (ends, missing pages) follow one
    // by one.  A branch between the two around the sums would have them copied.
    auto whole = [&](const NarrowPages &k, int T) {
        return k.page[0] >= 0 && k.page[1] >= 0 && T >= w.allLo && T + 32 <= w.allHi;
    };
    NarrowPages pages;
    int rest = end;  // the first tile that is not whole
    auto next_whole = [&](int T) {  // the wave's next whole tile from T on, its pages in `pages`; `end` if there is none
        for (; T < end; T += 128) {
            pages = narrow_pages<P>(p, s, T, w.anyLo, end);
            if (whole(pages, T)) return T;
            rest = min(rest, T);
        }
        return end;
    };
    NarrowTile<D> t0, t1;
    int T = next_whole(begin + 32 * (int)wave);
    const NarrowPages firstPages = pages;
    if (D < 256 && T < end) load_narrow<D, P>(t0, firstPages, p, h, T, n, g);
    int U = next_whole(T + 128);
    h8 qb[TERMS][D / 32];
    const float qf = load_query<D / 32, TERMS>(p.q + (size_t)c.row * p.qStride + (size_t)c.head * D, n < cols,
                                               p.scale, 16 * g, 64, 8, qb, column_max4);
    NarrowState<D> st = {};
    float vtop = 0.0f;
    st.m = ER_NO_MAX;
    if constexpr (D < 256) {
        while (T < end) {
            if (U < end) load_narrow<D, P>(t1, pages, p, h, U, n, g);
            T = next_whole(U + 128);
            attend_narrow<D, TERMS, false>(st, t0, qb, qf, 0, 0, 0, w, g, vtop);
            if (U >= end) break;
            if (T < end) load_narrow<D, P>(t0, pages, p, h, T, n, g);
            U = next_whole(T + 128);
            attend_narrow<D, TERMS, false>(st, t1, qb, qf, 0, 0, 0, w, g, vtop);
        }
    } else {
        // 16 KB a tile: one in registers, and twice the waves; the first waits
        // until the query's fp32 values have left theirs
        if (T < end) load_narrow<D, P>(t0, firstPages, p, h, T, n, g);
        while (T < end) {
            attend_narrow<D, TERMS, false>(st, t0, qb, qf, 0, 0, 0, w, g, vtop);
            T = U;
            if (T < end) load_narrow<D, P>(t0, pages, p, h, T, n, g);
            U = next_whole(T + 128);
        }
    }
    vtop = st.vref;  // it has only gone up
    bool second = false;  // of a tile whose halves' value scales lie far apart: a column may see the small one alone
    for (T = rest; T < end;) {
        pages = narrow_pages<P>(p, s, T, w.anyLo, end);
        if (!whole(pages, T) && (pages.page[0] >= 0 || pages.page[1] >= 0)) {
            load_narrow<D, P>(t0, pages, p, h, T, n, g);
            if constexpr (P < 32) {
                ScaleRange r = {0u, ~0u};
                r.add(__float_as_uint(uniform(t0.vs[0])));
                r.add(__float_as_uint(uniform(t0.vs[1])));
                if (pages.page[0] >= 0 && pages.page[1] >= 0 && r.apart()) {
                    t0.page[0] = second ? -1 : t0.page[0];
                    t0.page[1] = second ? t0.page[1] : -1;
                    second = !second;
                }
            }
            attend_narrow<D, TERMS, true>(st, t0, qb, qf, T, c.lo, c.hi, w, g, vtop);
        }
        if (!second) T += 128;
    }
    // each wave marks its own sums, for the tokens of all four: the sums are joined, and NaN is NaN in any of them
    if (__any(st.nans)) mark_nans<D>(st, p, s, h, begin, end, c.lo, c.hi, g);

    // the waves' columns, [wave][column][D + 4], and their references and sums (-1: nothing seen)
    constexpr uint32_t PITCH = D + 4;
    float *sm = lds + 64 * PITCH, *sl = sm + 64;
    const float l = column_sum4(st.l);
    const bool seen = column_max4(st.seen ? 1.0f : 0.0f) > 0.0f;
    if (n < cols) {
        float *at = lds + (wave * cols + n) * PITCH;
        const float f = st.vref * 0.0078125f * over(l);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 16; j += 4)
                *(f32x4 *)(at + (4 * g + i) * (D / 16) + j) =
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
        float f[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float l = sl[v * 16 + col];
            f[v] = l < 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f(sm[v * 16 + col] - m);
            visible |= !(l < 0.0f);
            total += f[v];
        }
        f32x4 o = {};
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (!(sl[v * 16 + col] < 0.0f)) o += *(const f32x4 *)(lds + (v * cols + col) * PITCH + d) * share_of(f[v], total);
        if (complete) {
            const Column k = column_of(p, q, h, col0 + col);
            store4(p, k.row, k.head, d, D, joined(o, visible, total));
        } else {
            const size_t at = (size_t)part * 16 + col;
            if (visible) *(f32x4 *)(p.partO + at * D + d) = o;
            if (d == 0) {
                p.partML[2 * at] = m;
                p.partML[2 * at + 1] = visible ? total : -1.0f;
            }
        }
    }
}

template <int D, int P, int TERMS>
ER_DEV void kv8_attend_narrow(const ErAttendArgs &p, float *lds) {
    const uint32_t H = p.c.heads, lane = threadIdx.x & 63u;
    if (p.shares == 0) {
        const uint32_t block = blockIdx.x % p.tiles, h = blockIdx.x / p.tiles % H, s = blockIdx.x / p.tiles / H;
        const LaneSequence l = lane_sequence(p, s);
        if (block < blocks_of(p, l.q)) narrow_unit<D, P, TERMS>(p, s, l.q, h, 16 * block, 0, l.steps, true, 0, lds);
        return;
    }
    const LaneSequence first = lane_sequence(p, lane);
    const Shares sh = shares_of(p, first, lane);
    uint32_t at = blockIdx.x * sh.quota;
    const uint32_t last = min(at + sh.quota, sh.total);
    if (at >= last) return;
    uint32_t begins, s = sequence_at(p, first, sh.aligned, at, lane, begins);
    LaneSequence l = lane_sequence_at(p, first, s);
    // Sequences behind the 64th are read again.  Should the batch's arrays change meanwhile,
    // the outputs mean nothing, but every workgroup ends and stays inside the buffers.
    if (l.steps == 0) return;
    uint32_t length = shared_length(p, l.steps, sh.aligned), unit = (at - begins) / length;
    if (unit >= H * blocks_of(p, l.q)) return;
    begins += unit * length;
    while (true) {
        // a unit that begins here and goes on in later workgroups leaves its
        // sums in this one's second part, one that began earlier in its first
        const uint32_t from = at - begins, to = min(last - begins, l.steps);
        const uint32_t blocks = blocks_of(p, l.q);
        narrow_unit<D, P, TERMS>(p, s, l.q, unit / blocks, unit % blocks * 16, from, to, from == 0 && to == l.steps,
                                 2 * blockIdx.x + (from == 0 ? 1u : 0u), lds);
        begins += length;
        at = begins;
        if (at >= last) return;
        if (++unit == H * blocks) {
            unit = 0;
            do {
                if (++s >= p.b.sequences) return;
                l = lane_sequence(p, s);
            } while (l.steps == 0);
            length = shared_length(p, l.steps, sh.aligned);
        }
        __syncthreads();  // the sums in LDS have been read
    }
}

// ---------------------------------------------------------------- many columns: prefill

#define ER_WIDE_TOKENS 64

// What a tile's pages bring: 64 / P of them.
template <int P>
struct WidePages {
    static constexpr int N = ER_WIDE_TOKENS / P;
    int page[N];
    float ks[N], vs[N];
};
// What the products need of them: a bit for each part that is there, and the scales (values' as integers, 0 where it is not).
template <int P>
struct WideParts {
    static constexpr uint32_t ALL = (1u << WidePages<P>::N) - 1u;
    uint32_t there, vs[WidePages<P>::N];
    float ks[WidePages<P>::N];
};
template <int P>
ER_DEV void parts_of(WideParts<P> &r, const WidePages<P> &w) {
    r.there = 0;
#pragma unroll
    for (int i = 0; i < w.N; ++i) {
        r.there |= (w.page[i] >= 0 ? 1u : 0u) << i;
        r.ks[i] = w.ks[i];
        r.vs[i] = w.page[i] >= 0 ? __float_as_uint(w.vs[i]) : 0u;
    }
}
template <int D, int P>
struct WideTile {
    u32x4 k[D / 64];                       // token tid / 4, bytes [(tid & 3) D/4, + D/4)
    uint32_t v[(D + 127) / 128][8];        // see value_item
};

// 64 entries of the page table with their scales, one a lane, and a tile's out
// of them by lane reads.  Loading them tile by tile into scalar registers would
// have every LDS wait of the tile wait for them too: scalar loads share its
// counter, and return out of order.
template <int P>
struct PageWindow {
    int first;  // table entry of lane 0
    int page;
    float ks, vs;
};
template <int P>
ER_DEV void fill_window(PageWindow<P> &w, const ErAttendArgs &p, uint32_t s, uint32_t h, int T, int lo, int end,
                        uint32_t lane) {
    const int tok = T + P * (int)lane;
    w.first = T / P;
    w.page = tok < end && tok + P > lo ? page_of(p.b, p.c, s, tok) : -1;
    const size_t block = (size_t)(uint32_t)max(w.page, 0) * p.c.heads + h;
    w.ks = p.c.ks[block];
    w.vs = p.c.vs[block];
}
// The pages of the tile at T; tiles are asked for in order.
template <int P>
ER_DEV WidePages<P> pages_at(PageWindow<P> &w, const ErAttendArgs &p, uint32_t s, uint32_t h, int T, int lo, int end,
                             uint32_t lane) {
    if (T / P - w.first >= 64) fill_window<P>(w, p, s, h, T, lo, end, lane);
    WidePages<P> r;
#pragma unroll
    for (int i = 0; i < r.N; ++i) {
        const int at = T / P - w.first + i;
        r.page[i] = __builtin_amdgcn_readlane(w.page, at);
        r.ks[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w.ks), at));
        r.vs[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w.vs), at));
    }
    return r;
}

// Entry of a tile's 16-token part, without an address (which would put v into scratch memory).
template <int N, typename T>
ER_DEV T of_part(const T (&v)[N], uint32_t part) {
    if constexpr (N == 1) {
        return v[0];
    } else if constexpr (N == 2) {
        const T a = v[0], b = v[1];
        return part & 2u ? b : a;
    } else {
        const T a = v[0], b = v[1], c = v[2], d = v[3];
        const T x = part & 1u ? b : a, y = part & 1u ? d : c;
        return part & 2u ? y : x;
    }
}

// Item `it` of a tile's values: four codes (dword) of the eight tokens (first
// .. first + 3, first + 8 .. first + 11) that one lane half holds of a
// 16-token slice of S^T.
struct ValueItem {
    uint32_t slot, dword, part;
    int first;
};
template <int D>
ER_DEV ValueItem value_item(uint32_t tid, uint32_t r) {
    const uint32_t it = (tid + ER_KV8_THREADS * r) & (2 * D - 1);  // D = 64: half the threads repeat
    ValueItem v;
    v.slot = it / (D / 4);
    v.dword = it % (D / 4);
    v.part = D >= 128 ? uniform(v.slot >> 1) : v.slot >> 1;  // from width 128 on the same for the wave
    v.first = (int)(16 * v.part + 4 * (v.slot & 1));
    return v;
}

template <int D, int P>
ER_DEV void load_wide(WideTile<D, P> &t, const WidePages<P> &w, const ErAttendArgs &p, uint32_t h, uint32_t tid) {
    {
        // a wave's 16 tokens are one part; the part's start is the same for the wave
        const uint32_t part = uniform(tid >> 6);
        const size_t block = (size_t)(uint32_t)max(of_part(w.page, part), 0) * p.c.heads + h;
        const uint8_t *src = p.c.k + block * (P * D) + (16 * part % P) * D;
        const uint32_t at = ((tid & 63u) >> 2) * D + (tid & 3u) * (D / 4);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) t.k[j] = *(const u32x4 *)(src + at + 16 * j);
    }
#pragma unroll
    for (int r = 0; r < (D + 127) / 128; ++r) {
        const ValueItem it = value_item<D>(tid, r);
        const size_t block = (size_t)(uint32_t)max(of_part(w.page, it.part), 0) * p.c.heads + h;
        const uint8_t *src = p.c.v + block * (P * D) + (16 * it.part % P) * D;
        const uint32_t at = 4 * (it.slot & 1) * D + 4 * it.dword;
#pragma unroll
        for (int i = 0; i < 8; ++i) t.v[r][i] = *(const uint32_t *)(src + at + ((i & 3) + 8 * (i >> 2)) * D);
    }
}

// A tile's codes in LDS: keys by token, values by element with the tokens of
// lane half hh's slice sl at bytes 32 hh + 8 sl, so that one 16-byte read holds
// the codes of two operands.  The pitches put consecutive rows 4 and 20 banks
// apart, which spreads 16 of them over all 64.
template <int D>
struct WideLds {
    uint8_t k[ER_WIDE_TOKENS][D + 16];
    uint8_t v[D][ER_WIDE_TOKENS + 16];
};

// The values of a tile that some column of the workgroup does not see whole,
// as attend_narrow's masked tiles; not 0 where there were NaN codes.
template <int D, int P>
ER_DEV uint32_t mask_wide(WideTile<D, P> &t, uint32_t there, int T, int lo, int hi, uint32_t tid) {
    uint32_t nan = 0;
#pragma unroll
    for (int r = 0; r < (D + 127) / 128; ++r) {
        const ValueItem it = value_item<D>(tid, r);
        const bool ok = there >> 16 * it.part / P & 1u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int tok = T + it.first + (i & 3) + 8 * (i >> 2);
            const uint32_t c = ok && tok >= lo && tok < hi ? t.v[r][i] : 0u, nans = nan_codes(c);
            nan |= nans;
            t.v[r][i] = c & ~nans;
        }
    }
    return nan;
}

// A tile into LDS.
template <int D, int P>
ER_DEV void store_wide(WideLds<D> &to, const WideTile<D, P> &t, uint32_t tid) {
    uint8_t *dst = &to.k[tid >> 2][(tid & 3u) * (D / 4)];
#pragma unroll
    for (int j = 0; j < D / 64; ++j) *(u32x4 *)(dst + 16 * j) = t.k[j];
#pragma unroll
    for (int r = 0; r < (D + 127) / 128; ++r) {
        const ValueItem it = value_item<D>(tid, r);
        const uint32_t *x = t.v[r];
        const uint32_t a0 = zip_lo(x[0], x[1]), a1 = zip_hi(x[0], x[1]), b0 = zip_lo(x[2], x[3]), b1 = zip_hi(x[2], x[3]);
        const uint32_t c0 = zip_lo(x[4], x[5]), c1 = zip_hi(x[4], x[5]), d0 = zip_lo(x[6], x[7]), d1 = zip_hi(x[6], x[7]);
        uint8_t *v = &to.v[4 * it.dword][32 * (it.slot & 1) + 8 * it.part];
        constexpr uint32_t PITCH = ER_WIDE_TOKENS + 16, LOW = 0x05040100u, HIGH = 0x07060302u;
        *(u32x2 *)v = u32x2{__builtin_amdgcn_perm(b0, a0, LOW), __builtin_amdgcn_perm(d0, c0, LOW)};
        *(u32x2 *)(v + PITCH) = u32x2{__builtin_amdgcn_perm(b0, a0, HIGH), __builtin_amdgcn_perm(d0, c0, HIGH)};
        *(u32x2 *)(v + 2 * PITCH) = u32x2{__builtin_amdgcn_perm(b1, a1, LOW), __builtin_amdgcn_perm(d1, c1, LOW)};
        *(u32x2 *)(v + 3 * PITCH) = u32x2{__builtin_amdgcn_perm(b1, a1, HIGH), __builtin_amdgcn_perm(d1, c1, HIGH)};
    }
}

ER_DEV float column_max2(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
ER_DEV float column_sum2(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// As the narrow kernel's.
template <int D>
ER_DEV void mark_nans(f32x16 (&o)[D / 32], const ErAttendArgs &p, uint32_t s, uint32_t h, int begin, int end, int lo,
                      int hi, uint32_t hh) {
    for (int tok = max(begin, lo); tok < min(end, hi); ++tok) {
        const int page = page_of(p.b, p.c, s, tok);
        if (page < 0) continue;
        const size_t slot = (((size_t)page * p.c.heads + h) << p.c.shift) + ((uint32_t)tok & ((1u << p.c.shift) - 1u));
        const uint8_t *v = p.c.v + slot * D;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t nan = nan_codes(*(const uint32_t *)(v + 32 * d + 8 * i + 4 * hh));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[d][4 * i + j] = (nan >> (8 * j)) & 1u ? __builtin_nanf("") : o[d][4 * i + j];
            }
    }
}

// 128 columns against one piece of their sequence's tokens, 32 columns a wave:
// bound by the matrix products and, nearly as much, by the instructions of the
// softmax and the conversions.  The four waves copy each 64-token tile's codes
// into LDS while the tile before is worked on, and convert them as they read
// operands: codes are half the LDS traffic of fp16, and leave more registers
// (fp16 in LDS spilled at head width 256).  A 4096-token prompt of an 8B layer
// (137 GFLOP) takes 187 to 193 us, up to 735 TFLOP/s, two waves a SIMD; ragged chunks behind
// long prefixes in fp32 (two terms, 35 GFLOP of products) 75 us with the join, and the
// prompt in fp32 270.
template <int D, int P, int TERMS>
ER_DEV void kv8_attend_wide(const ErAttendArgs &p, WideLds<D> *lds) {
    // One row tile of all units (sequence, piece, head) after the other, each
    // begun a sequence's heads later than the one before.  Workgroups go to the
    // 8 XCDs in turn: with 8 heads (or 16, ..) an XCD's L2 serves all tiles of a
    // head, with fewer a head's tiles lie on several, and units of very
    // different lengths load all XCDs alike.  Later tiles see more, and start first.
    const uint32_t units = p.b.sequences * p.splits * p.c.heads, round = blockIdx.x / units;
    const uint32_t ahead = round % (p.b.sequences * p.splits) * p.c.heads, at = blockIdx.x % units;
    const uint32_t unit = at >= ahead ? at - ahead : at + units - ahead, tile = p.tiles - 1 - round;
    const uint32_t h = unit % p.c.heads, piece = unit / p.c.heads % p.splits, s = unit / p.c.heads / p.splits;
    const Sequence q = sequence_of(p.b, s);
    const uint32_t cols = (uint32_t)q.n * p.group, col0 = tile * 128;
    if (col0 >= cols) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), n = lane & 31u, hh = lane >> 5;
    const Spans w = spans_of(p, q, col0, min(col0 + 127, cols - 1));
    const uint32_t wcol0 = col0 + 32 * wave;
    const bool idle = wcol0 >= cols;
    const Spans ww = spans_of(p, q, min(wcol0, cols - 1), min(wcol0 + 31, cols - 1));
    const Column c = column_of(p, q, h, min(wcol0 + n, cols - 1));
    const bool live = wcol0 + n < cols;
    const int begin = (w.anyLo & ~63) + (int)(piece * p.chunk), end = min(w.anyHi, begin + (int)p.chunk);

    f32x16 o[D / 32] = {};  // o[d][i]: value 32 d + (i & 3) + 8 (i >> 2) + 4 hh of column n, in units of vref / 128
    float m = ER_NO_MAX, l = 0.0f, vref = 0.0f, vinv = 0.0f, vtop = 0.0f;
    uint32_t seen = 0;  // not a mask, which would take two scalar registers
    if (begin < end) {
        WideTile<D, P> t;
        PageWindow<P> window;
        fill_window<P>(window, p, s, h, begin, w.anyLo, end, lane);
        // The next tile to load, and the one in `t`.  A tile that not all columns see
        // whole, and whose parts' value scales lie far apart, is taken part by part (`part`: a bit), since a column may see
        // the small ones alone.
        int next = begin, at = begin;
        uint32_t part = 0;
        WideParts<P> now;
        auto fetch = [&]() {
            at = next;
            if (next >= end) return;
            WidePages<P> pages = pages_at<P>(window, p, s, h, next, w.anyLo, end, lane);
            parts_of(now, pages);
            if constexpr (P < 64) {
                ScaleRange range = {0u, ~0u};
#pragma unroll
                for (int i = 0; i < pages.N; ++i) range.add(now.vs[i]);
                if (range.apart() && !(now.there == now.ALL && next >= w.allLo && next + 64 <= w.allHi)) {
                    part = max(part, 1u);
#pragma unroll
                    for (int i = 0; i < pages.N; ++i) pages.page[i] = part >> i & 1u ? pages.page[i] : -1;
                    parts_of(now, pages);
                    part = part <= now.ALL / 2 ? part << 1 : 0u;
                }
            }
            load_wide<D, P>(t, pages, p, h, tid);
            if (part == 0) next += 64;
        };
        fetch();
        h8 qb[TERMS][D / 16];
        const float qf = load_query<D / 16, TERMS>(p.q + (size_t)c.row * p.qStride + (size_t)c.head * D, live, p.scale,
                                                   16 * hh, 32, 8, qb, column_max2);
        uint32_t nans = 0;
        auto whole = [&](const WideParts<P> &k, const Spans &w, int T) {
            return k.there == k.ALL && T >= w.allLo && T + 64 <= w.allHi;
        };
        auto bring = [&](uint32_t to) {  // the tile in `t` into LDS
            if (!whole(now, w, at)) nans |= mask_wide<D, P>(t, now.there, at, w.anyLo, end, tid);
            store_wide<D, P>(lds[to], t, tid);
        };
        bring(0);
        int T = at;
        WideParts<P> parts = now;
        fetch();
        uint32_t buf = 0;
        // a wave without columns only brings its part of the tiles
        for (; idle && T < end; buf ^= 1u) {
            __syncthreads();
            if (at < end) bring(buf ^ 1u);
            T = at;
            fetch();
        }
        for (; T < end; buf ^= 1u) {
            __syncthreads();
            const WideLds<D> &in = lds[buf];
            const bool clear = whole(parts, ww, T);
            seen |= clear;
            ScaleRange range = {0u, ~0u};
#pragma unroll
            for (int i = 0; i < WidePages<P>::N; ++i) range.add(parts.vs[i]);
            follow_scale(range, vtop, vref, vinv, o);
#pragma unroll
            for (int th = 0; th < 2; ++th) {
                f32x16 sc = {};
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const u32x4 k = *(const u32x4 *)&in.k[32 * th + n][32 * j + 16 * hh];
                    const h8 a0 = codes_to_h8(k.x, k.y), a1 = codes_to_h8(k.z, k.w);
#pragma unroll
                    for (int term = 0; term < TERMS; ++term) {
                        sc = mfma32(a0, qb[term][2 * j], sc);
                        sc = mfma32(a1, qb[term][2 * j + 1], sc);
                    }
                }
                if (th == 1 && at < end) bring(buf ^ 1u);
                if (!clear) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int tok = T + 32 * th + 8 * (i >> 2) + 4 * (int)hh + (i & 3);
                        const bool shown = (parts.there >> (32 * th + 16 * (i >> 3)) / P & 1u) && tok >= c.lo && tok < c.hi;
                        seen |= shown ? 1u : 0u;
                        sc[i] = shown ? sc[i] : -__builtin_inff();
                    }
                }
                float f[2], v[2], top = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = (32 * th + 16 * i) / P;
                    const bool here = parts.there >> e & 1u;  // a missing part's values are zeros: any finite scale does
                    f[i] = score_factor(qf, here ? of_part(parts.ks, 2 * th + i) : 1.0f);
                    v[i] = here ? __uint_as_float(of_part(parts.vs, 2 * th + i)) * vinv : 1.0f;
                    float peak = sc[8 * i];
#pragma unroll
                    for (int j = 1; j < 8; ++j) peak = fmaxf(peak, sc[8 * i + j]);
                    top = fmaxf(top, peak * f[i]);
                }
                if (__any(top > m + ER_SLACK)) raise_reference(fmaxf(m, column_max2(top)), m, l, o);
                const float base = m - ER_LIFT;
                h8 wb[2][TERMS];
#pragma unroll
                for (int sl = 0; sl < 2; ++sl) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(sc[8 * sl + i] * f[sl] - base);
                    l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                    weight_terms<TERMS>(e, wb[sl]);
                }
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
                    const u32x4 x = *(const u32x4 *)&in.v[32 * d + n][32 * hh + 16 * th];
                    const h8 a0 = join(codes_to_h2<false>(x.x, v[0]), codes_to_h2<true>(x.x, v[0]),
                                       codes_to_h2<false>(x.y, v[0]), codes_to_h2<true>(x.y, v[0]));
                    const h8 a1 = join(codes_to_h2<false>(x.z, v[1]), codes_to_h2<true>(x.z, v[1]),
                                       codes_to_h2<false>(x.w, v[1]), codes_to_h2<true>(x.w, v[1]));
#pragma unroll
                    for (int term = 0; term < TERMS; ++term) {
                        o[d] = mfma32(a0, wb[0][term], o[d]);
                        o[d] = mfma32(a1, wb[1][term], o[d]);
                    }
                }
            }
            T = at;
            parts = now;
            fetch();
        }
        if (__syncthreads_or(nans != 0)) mark_nans<D>(o, p, s, h, begin, end, c.lo, c.hi, hh);
    }
    l = column_sum2(l);
    seen = column_max2(seen ? 1.0f : 0.0f) > 0.0f ? 1u : 0u;
    if (!live) return;
    const float f = p.splits == 1 ? vref * 0.0078125f / l : vref * 0.0078125f * over(l);
    const size_t to = part_index(p, piece, c.row, c.head);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at = 32 * d + 8 * i + 4 * hh;
            const f32x4 v = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * f;
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

ER_DEV float wave_top(float v) {
    v = dpp_max<ER_DPP_QUAD_XOR1>(v);
    v = dpp_max<ER_DPP_QUAD_XOR2>(v);
    v = dpp_max<ER_DPP_ROW_HALF_MIRROR>(v);
    v = dpp_max<ER_DPP_ROW_MIRROR>(v);
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16 * i));
    return fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
}

// One column's parts: weights l 2^(m - max) / sum from the references and sums,
// then the weighted outputs, D / 4 lanes a part.  index(i): where part i lies.
template <int D, typename INDEX>
ER_DEV void join_parts(const ErAttendArgs &p, uint32_t parts, int row, uint32_t head, float *lds, INDEX index) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    float *red = lds, *weight = lds + 4 * ER_KV8_THREADS;  // [lanes][4], [parts]
    float top = ER_NO_MAX;
    for (uint32_t i = lane; i < parts; i += 64) top = fmaxf(top, p.partML[2 * index(i)]);
    top = wave_top(top);
    float total = 0.0f;
    bool seen = false;
    for (uint32_t i = lane; i < parts; i += 64) {
        const size_t at = 2 * index(i);
        const float l = p.partML[at + 1];
        const bool some = !(l < 0.0f);
        const float f = some ? l * __builtin_amdgcn_exp2f(p.partML[at] - top) : -1.0f;
        if (some) total += f;
        seen |= some;
        if (tid < 64) weight[i] = f;
    }
    // every wave has the sum, of the same terms in the same order
    total = group_sum<64>(total);
    seen = __any(seen);
    for (uint32_t i = tid; i < parts && tid < 64; i += 64)
        if (!(weight[i] < 0.0f)) weight[i] = share_of(weight[i], total);
    __syncthreads();
    constexpr uint32_t LANES = D / 4, AT_ONCE = ER_KV8_THREADS / LANES;
    const uint32_t mine = tid / LANES, d = (tid % LANES) * 4;
    f32x4 o = {};
#pragma unroll 4
    for (uint32_t i = mine; i < parts; i += AT_ONCE) {
        const float f = weight[i];
        if (f >= 0.0f || f != f) o += *(const f32x4 *)(p.partO + index(i) * D + d) * f;
    }
    *(f32x4 *)(red + 4 * tid) = o;
    __syncthreads();
    if (tid < LANES) {
        f32x4 v = {};
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; ++k) v += *(const f32x4 *)(red + 4 * (k * LANES + tid));
        store4(p, row, head, 4 * tid, D, joined(v, seen, total));
    }
}

// One row and query head after the wide kernel (a part a piece) or the narrow
// one (a part a workgroup that had some of the unit's steps): 9 us for 64 users
// of 32 heads, 7 for one of 64 parts, a launch and a chain of loads.
template <int D>
ER_DEV void kv8_join(const ErAttendArgs &p, float *lds) {
    const uint32_t heads = p.group * p.c.heads, row = blockIdx.x / heads, head = blockIdx.x % heads;
    const uint32_t lane = threadIdx.x & 63u;
    const LaneSequence first = lane_sequence(p, lane);
    const uint32_t s = uniform(sequence_of_row(p.b, row, lane));
    if (s >= p.b.sequences) return;
    const LaneSequence l = lane_sequence_at(p, first, s);
    const Sequence &q = l.q;
    if ((int)row < q.row0 || (int)row >= q.row0 + q.n) return;
    if (p.shares == 0) {
        join_parts<D>(p, p.splits, (int)row, head, lds, [&](uint32_t i) { return part_index(p, i, (int)row, head); });
        return;
    }
    const Shares sh = shares_of(p, first, lane);
    uint32_t before = lane < s ? shared_length(p, first.steps, sh.aligned) * blocks_of(p, first.q) : 0;
    for (uint32_t i = 64 + lane; i < s; i += 64) {
        const LaneSequence b = lane_sequence(p, i);
        before += shared_length(p, b.steps, sh.aligned) * blocks_of(p, b.q);
    }
    before = wave_sum(before) * p.c.heads;
    const uint32_t col = (row - (uint32_t)q.row0) * p.group + head % p.group;
    const uint32_t unit = head / p.group * blocks_of(p, q) + (col >> 4);
    const uint32_t begins = before + unit * shared_length(p, l.steps, sh.aligned);
    const uint32_t w0 = begins / sh.quota, parts = (begins + l.steps - 1) / sh.quota - w0 + 1;
    if (parts == 1) return;  // one workgroup had it all and wrote it
    if (w0 + parts > p.shares) return;  // as in kv8_attend_narrow
    join_parts<D>(p, parts, (int)row, head, lds, [&](uint32_t i) {
        return (size_t)(2 * (w0 + i) + (i == 0 ? 1u : 0u)) * 16 + (col & 15u);
    });
}

// All heads of one row after the wide kernel, where the parts are few: four
// values a thread, its column's references and sums read by all its lanes.  Eight
// parts of 1033 rows of 14 heads of 64 take 9 us; a workgroup a column took 24 for five.
template <int D>
ER_DEV void kv8_join_row(const ErAttendArgs &p) {
    const uint32_t row = blockIdx.x, heads = p.group * p.c.heads, lane = threadIdx.x & 63u;
    const uint32_t s = uniform(sequence_of_row(p.b, row, lane));
    if (s >= p.b.sequences) return;
    const Sequence q = sequence_of(p.b, s);
    if ((int)row < q.row0 || (int)row >= q.row0 + q.n) return;
    for (uint32_t at = threadIdx.x; at < heads * (D / 4); at += ER_KV8_THREADS) {
        const uint32_t head = at / (D / 4), d = (at % (D / 4)) * 4;
        // all parts' references and sums at once
        float m[ER_KV8_ROW_PARTS], l[ER_KV8_ROW_PARTS], top = ER_NO_MAX, total = 0.0f;
        bool seen = false;
#pragma unroll
        for (uint32_t i = 0; i < ER_KV8_ROW_PARTS; ++i) {
            const f32x2 ml = i < p.splits ? *(const f32x2 *)(p.partML + 2 * part_index(p, i, (int)row, head)) : f32x2{ER_NO_MAX, -1.0f};
            m[i] = ml.x;
            l[i] = ml.y;
            top = fmaxf(top, ml.x);
        }
#pragma unroll
        for (uint32_t i = 0; i < ER_KV8_ROW_PARTS; ++i) {
            const bool some = !(l[i] < 0.0f);
            l[i] = some ? l[i] * __builtin_amdgcn_exp2f(m[i] - top) : -1.0f;
            total += some ? l[i] : 0.0f;
            seen |= some;
        }
        const float inverse = over(total);
        f32x4 o = {};
#pragma unroll
        for (uint32_t i = 0; i < ER_KV8_ROW_PARTS; ++i)
            if (i < p.splits && !(l[i] < 0.0f))
                o += *(const f32x4 *)(p.partO + part_index(p, i, (int)row, head) * D + d) * (l[i] * inverse);
        store4(p, (int)row, head, d, D, joined(o, seen, total));
    }
}

extern __shared__ __attribute__((aligned(16))) float er_kv8_lds[];

// One kernel for each head width, page size and output type.  WAVES: waves a
// SIMD that the registers leave room for.
#define ER_KV8_NARROW(D, P, TERMS, NAME, WAVES)                                                                    \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS, WAVES)                                            \
        er_kv8_attend_narrow_d##D##_p##P##_##NAME(ErAttendArgs p) {                                                \
        __shared__ __attribute__((aligned(16))) float sums[64 * (D + 4) + 128];                                    \
        kv8_attend_narrow<D, P, TERMS>(p, sums);                                                                   \
    }
#define ER_KV8_WIDE(D, P, TERMS, NAME, WAVES)                                                                      \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS, WAVES)                                            \
        er_kv8_attend_wide_d##D##_p##P##_##NAME(ErAttendArgs p) {                                                  \
        __shared__ __attribute__((aligned(16))) WideLds<D> tiles[2];                                               \
        kv8_attend_wide<D, P, TERMS>(p, tiles);                                                                    \
    }
#define ER_KV8_PAGES(D, P, NARROW, WIDE)                                                                           \
    ER_KV8_NARROW(D, P, 1, bf16, 2)                                                                                \
    ER_KV8_NARROW(D, P, 2, f32, NARROW)                                                                            \
    ER_KV8_WIDE(D, P, 1, bf16, WIDE)                                                                               \
    ER_KV8_WIDE(D, P, 2, f32, WIDE)
#define ER_KV8_ATTEND(D, WIDE) ER_KV8_PAGES(D, 32, 2, WIDE) ER_KV8_PAGES(D, 64, 2, WIDE)
ER_KV8_ATTEND(64, 3)
ER_KV8_ATTEND(128, 2)
ER_KV8_ATTEND(256, 1)
ER_KV8_PAGES(64, 16, 2, 3)
ER_KV8_PAGES(128, 16, 2, 2)
// two pages a tile, two terms and wide heads need a few registers over the 256 that two waves leave
ER_KV8_PAGES(256, 16, 1, 1)

#define ER_KV8_JOIN(D)                                                                                             \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS) er_kv8_join_d##D(ErAttendArgs p) {                \
        kv8_join<D>(p, er_kv8_lds);                                                                                \
    }                                                                                                              \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS) er_kv8_join_row_d##D(ErAttendArgs p) {            \
        kv8_join_row<D>(p);                                                                                        \
    }
ER_KV8_JOIN(64)
ER_KV8_JOIN(128)
ER_KV8_JOIN(256)
