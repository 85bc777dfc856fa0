// er_kv8.hip -- what stands between the q/k/v and the output projections: head
// norms with the position rotation, appends to a paged cache of e4m3 codes,
// and attention over it.  A code object of its own, compiled beside
// er_kernels.hip's.
#include "er_common.h"
#include "er_kv8.h"

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

// A value that every lane holds alike, moved to a scalar register.
ER_DEV uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
ER_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
ER_DEV float uniform(float v) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

// A value that no kernel of the launch writes, at an address that all lanes
// share: a scalar load, which waits for no vector load in flight.
template <typename T>
ER_DEV T load_shared(const T *p) {
    return *(const __attribute__((address_space(4))) T *)(uintptr_t)p;
}

// ---------------------------------------------------------------- rows of a batch

// Sequence s as the kernels see it: whatever the device arrays hold, rows stay
// inside the row buffers and tokens inside the page table.
struct Sequence {
    int row0, n, len;  // first row, rows, tokens
};
ER_DEV Sequence sequence_of(const ErKv8Batch &b, uint32_t s) {
    const int rows = (int)b.rows;
    Sequence q;
    q.row0 = min(max(load_shared(b.start + s), 0), rows);
    q.n = min(max(min(load_shared(b.start + s + 1), rows) - q.row0, 0), (int)b.maxRows);
    q.len = min(max(load_shared(b.len + s), 0), (int)b.maxLen);
    return q;
}

// The page that token t (0 <= t < len) of sequence s lies in, or -1.
ER_DEV int page_of(const ErKv8Batch &b, const ErKv8Cache &c, uint32_t s, int t) {
    const int p = load_shared(b.table + (size_t)s * b.stride + ((uint32_t)t >> c.shift));
    return (uint32_t)p < c.pages ? p : -1;
}

// ---------------------------------------------------------------- norm and rotation

// Eight values of a head, as four pairs that turn together.  Lane `sub` of the
// head's D / 8 lanes holds pairs 4 sub .. 4 sub + 3.  Pairs behind the rotated
// ones are neighbours, whatever the order of the rotated ones, so that the
// D / 2 pairs cover the head.
struct Pairs {
    float a[4], b[4];
};
// Element that a[0] is read from; b[0] is `apart` elements on; neighbours
// interleave (a[i], b[i] at 2 i, 2 i + 1), halves do not.
struct PairPlace {
    uint32_t at, apart;
    bool neighbours, turns;
};
ER_DEV PairPlace pair_place(uint32_t sub, uint32_t rot, uint32_t pairs) {
    PairPlace p;
    p.turns = 8u * sub < rot;
    p.neighbours = pairs || !p.turns;
    p.at = p.neighbours ? 8u * sub : 4u * sub;
    p.apart = p.neighbours ? 4u : rot / 2u;
    return p;
}
// The choices are made on values: choosing between elements of a vector would
// index it at run time, through memory.
ER_DEV float choose(bool c, float x, float y) { return c ? x : y; }
ER_DEV Pairs to_pairs(f32x4 lo, f32x4 hi, bool neighbours) {
    Pairs v;
    v.a[0] = lo.x;
    v.a[1] = choose(neighbours, lo.z, lo.y);
    v.a[2] = choose(neighbours, hi.x, lo.z);
    v.a[3] = choose(neighbours, hi.z, lo.w);
    v.b[0] = choose(neighbours, lo.y, hi.x);
    v.b[1] = choose(neighbours, lo.w, hi.y);
    v.b[2] = choose(neighbours, hi.y, hi.z);
    v.b[3] = hi.w;
    return v;
}
ER_DEV void from_pairs(const Pairs &v, bool neighbours, f32x4 &lo, f32x4 &hi) {
    lo = f32x4{v.a[0], choose(neighbours, v.b[0], v.a[1]), choose(neighbours, v.a[1], v.a[2]),
               choose(neighbours, v.b[1], v.a[3])};
    hi = f32x4{choose(neighbours, v.a[2], v.b[0]), choose(neighbours, v.b[2], v.b[1]),
               choose(neighbours, v.a[3], v.b[2]), v.b[3]};
}
ER_DEV Pairs load_pairs(const float *p, const PairPlace &pl) {
    const f32x4 lo = *(const f32x4_a4 *)(p + pl.at);
    const f32x4 hi = *(const f32x4_a4 *)(p + pl.at + pl.apart);
    return to_pairs(lo, hi, pl.neighbours);
}

// cos and sin of a fraction of a turn, |x| <= 1/2.  The nearest quarter turn is taken off
// exactly, in 64 bits, and the angle that is left, |a| <= pi / 4, rounded once
// to fp32 (2^-25); the Taylor series end where their next terms are below
// 2^-28 (a^11 / 11! and a^12 / 12!).  At most 7e-8 off; about half the
// instructions of two library calls, which reduce each on its own.
ER_DEV void cos_sin_turn(double x, float &c, float &s) {
    const double q = rint(4.0 * x);
    const float a = (float)((x - 0.25 * q) * 6.283185307179586477), z = a * a;
    float sn = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    sn = __builtin_fmaf(z, sn, 8.3333333e-3f);
    sn = __builtin_fmaf(z, sn, -1.6666667e-1f);
    sn = __builtin_fmaf(a * z, sn, a);
    float cs = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    cs = __builtin_fmaf(z, cs, -1.3888889e-3f);
    cs = __builtin_fmaf(z, cs, 4.1666667e-2f);
    cs = __builtin_fmaf(z, cs, -0.5f);
    cs = __builtin_fmaf(z, cs, 1.0f);
    const int k = (int)q;
    const float u = k & 1 ? sn : cs, v = k & 1 ? cs : sn;
    c = (k + 1) & 2 ? -u : u;
    s = k & 2 ? -v : v;
}

// The four pairs' frequencies in turns, and their cos and sin at a position.
// position * frequency is formed and reduced in 64 bits (at position 10^6 an
// fp32 product is off by 0.03 rad).
struct Frequencies {
    double f[4];
    bool on;
};
struct Turns {
    float c[4], s[4];
    bool on;
};
ER_DEV Frequencies frequencies_of(const float *freq, uint32_t sub, bool turns) {
    Frequencies r = {};
    r.on = turns;
    if (turns) {
        const f32x4 f = *(const f32x4_a4 *)(freq + 4u * sub);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.f[i] = (double)f[i] * 0.15915494309189533577;  // 1 / 2 pi
    }
    return r;
}
ER_DEV Turns turns_of(int position, const Frequencies &f) {
    Turns t = {};
    t.on = f.on;
    if (f.on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double turn = (double)position * f.f[i];
            cos_sin_turn(turn - rint(turn), t.c[i], t.s[i]);
        }
    }
    return t;
}

template <int CTRL>
ER_DEV double dpp_of(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int W>
ER_DEV double group_sum64(double v) {  // W = 8, 16 or 32 lanes
    v += dpp_of<ER_DPP_QUAD_XOR1>(v);
    v += dpp_of<ER_DPP_QUAD_XOR2>(v);
    v += dpp_of<ER_DPP_ROW_HALF_MIRROR>(v);
    if constexpr (W >= 16) v += dpp_of<ER_DPP_ROW_MIRROR>(v);
    if constexpr (W == 32) v += __shfl_xor(v, 16);
    return v;
}
// 1 / sqrt of the mean of a head's D squares plus eps; `sum` is this lane's part
// of the sum.  In 64 bits, where the squares of no fp32 values leave the range. One Newton
// step doubles the correct bits of the instruction's root, over 20.
template <int D>
ER_DEV double head_rsqrt(double sum, double eps) {
    const double ms = group_sum64<D / 8>(sum) * (1.0 / D) + eps, r0 = __builtin_amdgcn_rsq(ms);
    return ms < __builtin_inf() ? r0 * __builtin_fma(-0.5 * ms * r0, r0, 1.5) : r0;
}

// The head's values normed (w: this lane's norm weights) and rotated.  D / 8
// lanes hold the head, so its sum of squares is a sum over that lane group.
template <int D>
ER_DEV void norm_turn(Pairs &v, bool norm, const Pairs &w, const Turns &t, float eps) {
    if (norm) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a = (double)v.a[i], b = (double)v.b[i];
            sum = __builtin_fma(b, b, __builtin_fma(a, a, sum));
        }
        const double r = head_rsqrt<D>(sum, (double)eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v.a[i] = (float)((double)v.a[i] * r) * w.a[i];
            v.b[i] = (float)((double)v.b[i] * r) * w.b[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // a pair that does not turn passes as it is (its partner may be infinite)
        const float a = v.a[i], b = v.b[i];
        v.a[i] = t.on ? a * t.c[i] - b * t.s[i] : a;
        v.b[i] = t.on ? b * t.c[i] + a * t.s[i] : b;
    }
}

// The same in 64 bits for keys on their way into codes: rounded to fp32 before,
// one in some hundred thousand, those next to a border, would get the other
// code.  64-bit operations run at the rate of 32-bit ones here (the fp32 form
// took 14 us for three ragged prompts of an 8B layer, this one 16); the
// results go to fp32 by rounding to odd, which no later rounding to fewer bits
// notices.
ER_DEV float round_to_odd(double v) {
    float f = (float)v;
    const double back = (double)f;
    uint32_t u = __float_as_uint(f);
    if (fabs(back) > fabs(v)) u -= 1;  // to zero
    if (back != v && v == v) u |= 1;
    return __uint_as_float(u);
}
// cos and sin of a fraction of a turn as cos_sin_turn; the next terms of the
// series are below 2^-40.
ER_DEV void cos_sin_turn64(double x, double &c, double &s) {
    const double q = rint(4.0 * x);
    const double a = (x - 0.25 * q) * 6.283185307179586477, z = a * a;
    double sn = __builtin_fma(z, 1.6059043836821613e-10, -2.5052108385441719e-8);
    sn = __builtin_fma(z, sn, 2.7557319223985893e-6);
    sn = __builtin_fma(z, sn, -1.9841269841269841e-4);
    sn = __builtin_fma(z, sn, 8.3333333333333333e-3);
    sn = __builtin_fma(z, sn, -1.6666666666666667e-1);
    sn = __builtin_fma(a * z, sn, a);
    double cs = __builtin_fma(z, 2.0876756987868099e-9, -2.7557319223985891e-7);
    cs = __builtin_fma(z, cs, 2.4801587301587302e-5);
    cs = __builtin_fma(z, cs, -1.3888888888888889e-3);
    cs = __builtin_fma(z, cs, 4.1666666666666667e-2);
    cs = __builtin_fma(z, cs, -0.5);
    cs = __builtin_fma(z, cs, 1.0);
    const int k = (int)q;
    const double u = k & 1 ? sn : cs, v = k & 1 ? cs : sn;
    c = (k + 1) & 2 ? -u : u;
    s = k & 2 ? -v : v;
}
struct Turns64 {
    double c[4], s[4];
};
ER_DEV void turns64_of(Turns64 &t, int position, const Frequencies &f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double turn = (double)position * f.f[i];
        cos_sin_turn64(turn - rint(turn), t.c[i], t.s[i]);
    }
}
// t further on by the angles of `by`.
ER_DEV void turn_on(Turns64 &t, const Turns64 &by) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double c = t.c[i] * by.c[i] - t.s[i] * by.s[i];
        t.s[i] = t.s[i] * by.c[i] + t.c[i] * by.s[i];
        t.c[i] = c;
    }
}
template <int D>
ER_DEV void norm_turn64(Pairs &p, bool norm, const Pairs &w, bool turns, const Turns64 &t, double eps) {
    double a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = (double)p.a[i];
        b[i] = (double)p.b[i];
    }
    if (norm) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __builtin_fma(b[i], b[i], __builtin_fma(a[i], a[i], sum));
        const double r = head_rsqrt<D>(sum, eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] *= r * (double)w.a[i];
            b[i] *= r * (double)w.b[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p.a[i] = round_to_odd(turns ? a[i] * t.c[i] - b[i] * t.s[i] : a[i]);
        p.b[i] = round_to_odd(turns ? b[i] * t.c[i] + a[i] * t.s[i] : b[i]);
    }
}

// One row's heads of one kind in strips of 512 / D, of which this wave takes
// chunk, chunk + chunks, ...: D / 8 lanes a head.
template <int D>
ER_DEV void turn_heads(const ErTurn &h, uint32_t row, uint32_t chunk, uint32_t chunks, uint32_t group,
                       const PairPlace &pl, const Turns &t, float eps) {
    constexpr uint32_t PER = 512 / D;
    const uint32_t strips = (h.heads + PER - 1) / PER;
    const uint32_t passes = strips > chunk ? (strips - chunk + chunks - 1) / chunks : 0;
    const bool norm = h.norm != nullptr;
    Pairs w = {};
    if (norm) w = load_pairs(h.norm, pl);
    const float *in = h.in + (size_t)row * h.inStride;
    float *out = h.out + (size_t)row * h.outStride;
    for (uint32_t i = 0; i < passes; ++i) {
        const uint32_t head = (i * chunks + chunk) * PER + group;
        const bool live = head < h.heads;
        Pairs v = {};
        if (live) v = load_pairs(in + (size_t)head * D, pl);
        norm_turn<D>(v, norm, w, t, eps);
        if (live) {
            f32x4 lo, hi;
            from_pairs(v, pl.neighbours, lo, hi);
            *(f32x4_a4 *)(out + (size_t)head * D + pl.at) = lo;
            *(f32x4_a4 *)(out + (size_t)head * D + pl.at + pl.apart) = hi;
        }
    }
}

// RMS norm and rotation of query and key heads: bytes in and out bound it.
// One wave takes every chunks-th strip of 512 / D heads of one row, so the
// row's angles (64-bit products, a sine and a cosine for every pair) are
// formed once for all of them.  All of a head's loads precede its stores and no
// other lane reads the head, so an output may be its own input.  4096 rows of 32
// + 8 heads of 128 take 38.3 us: 4.38 TB/s in and out, where a copy of as much
// reaches 4.7; one row 3.0 us, a launch.
template <int D>
ER_DEV void qk_norm_rope(const ErRopeArgs &p) {
    const uint32_t wave = uniform((blockIdx.x * ER_KV8_THREADS + threadIdx.x) >> 6);
    const uint32_t row = wave / p.chunks, chunk = wave - row * p.chunks;
    if (row >= p.rows) return;
    const uint32_t lane = threadIdx.x & 63u, sub = lane % (D / 8), group = lane / (D / 8);
    const PairPlace pl = pair_place(sub, p.rot, p.pairs);
    const Turns t = turns_of(p.positions ? p.positions[row] : 0, frequencies_of(p.freq, sub, pl.turns));
    constexpr uint32_t PER = 512 / D;
    // strips of the query heads, then of the key heads, dealt to the row's waves in turn
    const uint32_t qStrips = (p.q.heads + PER - 1) / PER;
    turn_heads<D>(p.q, row, chunk, p.chunks, group, pl, t, p.eps);
    turn_heads<D>(p.k, row, (chunk + p.chunks - qStrips % p.chunks) % p.chunks, p.chunks, group, pl, t, p.eps);
}

// ---------------------------------------------------------------- append

// log2 of the smallest power of two, from 2^-100 on, that brings a finite
// magnitude to at most 448 = 0.875 * 2^9.
ER_DEV int block_exponent(float peak) {
    const uint32_t u = __float_as_uint(peak);
    const int e = (int)(u >> 23) - 126;  // peak = m * 2^e, m in [0.5, 1)
    const int j = e - ((u & 0x7fffffu) <= 0x600000u ? 9 : 8);
    return max(j, -100);
}
ER_DEV float exp2i(int j) { return __uint_as_float((uint32_t)(j + 127) << 23); }

ER_DEV float finite_magnitude(float v) {
    const float m = fabsf(v);
    return m < __builtin_inff() ? m : 0.0f;  // NaN too
}

// Four values to e4m3 codes, nearest even.  Scaled values reach 448 at the
// most; infinities become NaN first, as the code has none.
ER_DEV float no_inf(float v) { return fabsf(v) == __builtin_inff() ? __builtin_nanf("") : v; }
ER_DEV uint32_t codes4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(no_inf(a), no_inf(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(no_inf(c), no_inf(d), r, true);
}
// Four codes times a power of two up to 1, to nearest even.
ER_DEV uint32_t recode4(uint32_t c, float f) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    return codes4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
}

ER_DEV float wave_max(float v) {
    v = dpp_max_nonneg<ER_DPP_QUAD_XOR1>(v);
    v = dpp_max_nonneg<ER_DPP_QUAD_XOR2>(v);
    v = dpp_max_nonneg<ER_DPP_ROW_HALF_MIRROR>(v);
    v = dpp_max_nonneg<ER_DPP_ROW_MIRROR>(v);
    const float a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0));
    const float b = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16));
    const float c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32));
    const float d = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 48));
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// The sequence that a row belongs to: how many of them end at or before it
// (the batch's `sequences` for a row behind the last).
ER_DEV uint32_t sequence_of_row(const ErKv8Batch &b, uint32_t row, uint32_t lane) {
    uint32_t s = 0;
    for (uint32_t at = 0; at < b.sequences; at += 64) {
        const bool behind = at + lane < b.sequences && b.start[at + lane + 1] <= (int)row;
        s += (uint32_t)__popcll(__ballot(behind));
    }
    return s;
}

template <int D>
ER_DEV void turn_query_row(const ErAppendArgs &p) {
    const uint32_t lane = threadIdx.x & 63u, sub = lane % (D / 8), group = lane / (D / 8);
    const uint32_t wave = uniform(((blockIdx.x - p.cacheBlocks) * ER_KV8_THREADS + threadIdx.x) >> 6);
    const uint32_t row = wave / p.chunks, chunk = wave - row * p.chunks;
    if (row >= p.b.rows) return;
    const uint32_t s = uniform(sequence_of_row(p.b, row, lane));
    if (s >= p.b.sequences) return;
    const Sequence q = sequence_of(p.b, s);
    const int at = (int)row - q.row0, position = q.len - q.n + at;
    if (at < 0 || at >= q.n || position < 0) return;
    const PairPlace pl = pair_place(sub, p.rot, p.pairs);
    const Turns t = turns_of(position, frequencies_of(p.freq, sub, pl.turns));
    turn_heads<D>(p.q, row, chunk, p.chunks, group, pl, t, p.eps);
}

// Appends to one block: the tokens of one page and head, keys or values.  One
// workgroup holds the block's new values in registers (at most 64 a lane), so
// that they are read once: their largest magnitude gives the scale, then they
// are coded.  Old codes are read only where the scale grows, and since scales
// are powers of two, growing one costs them nothing but subnormals.  No other
// workgroup touches the block, so nothing is ordered between workgroups.
// Three ragged prompts of an 8B layer (43 MB in and out, 9 us at a copy's rate)
// take 16 us: 2.3 of it are the keys' 64-bit rotations, which the workgroup of every
// head forms again, and the rest over the copy a workgroup's own chain, in which loads, norm,
// maximum and stores follow each other; a token of each of 64 users
// 5.8 us, bound by the chain start, table, scale, row.
template <int D, int P>
ER_DEV void append_block(const ErAppendArgs &p, float *peaks) {
    constexpr int LANES = D / 8;                                    // lanes a token
    constexpr int TOKENS = ER_KV8_THREADS / LANES < P ? ER_KV8_THREADS / LANES : P;  // tokens a pass
    constexpr int PASSES = P / TOKENS;
    const uint32_t H = p.c.heads;
    // keys first, as they take longer, and so that every XCD gets as many
    const bool values = blockIdx.x >= p.cacheBlocks / 2;
    uint32_t at = values ? blockIdx.x - p.cacheBlocks / 2 : blockIdx.x;
    const uint32_t head = at % H;
    at /= H;
    const uint32_t span = at % p.spans, s = at / p.spans;
    const Sequence q = sequence_of(p.b, s);
    const int first = max(q.len - q.n, 0);
    const int begin = (first / P + (int)span) * P;  // the page's first token
    if (q.n == 0 || begin >= q.len) return;
    const int t0 = max(first, begin), t1 = min(q.len, begin + P);
    const int page = uniform(page_of(p.b, p.c, s, begin));
    if (page < 0) return;
    const size_t block = (size_t)page * H + head;
    uint8_t *codes = (values ? p.c.v : p.c.k) + block * (size_t)(P * D);
    float *scale = (values ? p.c.vs : p.c.ks) + block;

    const uint32_t tid = threadIdx.x, sub = tid % LANES;
    const int slot = (int)(tid / LANES);
    // values take no rotation: their pairs are neighbours and stay
    const PairPlace pl = pair_place(sub, values ? 0u : p.rot, p.pairs);
    const bool norm = !values && p.kNorm != nullptr;
    Pairs w = {};
    if (norm) w = load_pairs(p.kNorm, pl);
    const Frequencies freq = frequencies_of(p.freq, sub, pl.turns);
    Turns64 turns = {}, onward = {};
    bool turned = false;
    Pairs v[PASSES];
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int t = begin + i * TOKENS + slot;
        const bool live = slot < TOKENS && t >= t0 && t < t1;
        v[i] = {};
        if (live) {
            const size_t row = (size_t)(q.row0 + q.n - (q.len - t));
            if (!values) {
                v[i] = load_pairs(p.k + row * p.kStride + (size_t)head * D, pl);
            } else if (p.vHalf) {
                const u16x4_a2 *h = (const u16x4_a2 *)((const uint16_t *)p.v + row * p.vStride + (size_t)head * D + pl.at);
                const u16x4_a2 l = h[0], u = h[1];
                v[i] = to_pairs(f32x4{f16_to_f32(l.x), f16_to_f32(l.y), f16_to_f32(l.z), f16_to_f32(l.w)},
                                f32x4{f16_to_f32(u.x), f16_to_f32(u.y), f16_to_f32(u.z), f16_to_f32(u.w)}, true);
            } else {
                v[i] = load_pairs((const float *)p.v + row * p.vStride + (size_t)head * D, pl);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int t = begin + i * TOKENS + slot;
        // passes without a new token are skipped by all lanes: a decode step's
        // block has one; from one pass to the next the angles grow by the same
        const int from = begin + i * TOKENS;
        if (!values && from < t1 && from + TOKENS > t0 && (norm || p.rot)) {
            if (p.rot) {
                if (!turned) {
                    turns64_of(turns, t, freq);
                    if (from + TOKENS < t1) turns64_of(onward, TOKENS, freq);
                    turned = true;
                } else {
                    turn_on(turns, onward);
                }
            }
            norm_turn64<D>(v[i], norm, w, freq.on, turns, (double)p.eps);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            peak = fmaxf(peak, fmaxf(finite_magnitude(v[i].a[e]), finite_magnitude(v[i].b[e])));
    }
    peak = wave_max(peak);
    if ((tid & 63u) == 0) peaks[tid >> 6] = peak;
    const float old = t0 > begin ? *scale : 0.0f;  // a page's first token finds whatever an earlier user left
    __syncthreads();
    peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
    const float need = exp2i(block_exponent(peak));
    const float now = fmaxf(old, need);
    if (now > old && t0 > begin) {
        const float f = old / now;
        for (uint32_t i = tid; i < (uint32_t)(t0 - begin) * (D / 4); i += ER_KV8_THREADS) {
            uint32_t *c = (uint32_t *)codes + i;
            *c = recode4(*c, f);
        }
    }
    const float f = 1.0f / now;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int t = begin + i * TOKENS + slot;
        const bool live = slot < TOKENS && t >= t0 && t < t1;
        if (!live) continue;
        f32x4 lo, hi;
        from_pairs(v[i], pl.neighbours, lo, hi);
        uint8_t *c = codes + (size_t)(t - begin) * D + pl.at;
        *(uint32_t *)c = codes4(lo.x * f, lo.y * f, lo.z * f, lo.w * f);
        *(uint32_t *)(c + pl.apart) = codes4(hi.x * f, hi.y * f, hi.z * f, hi.w * f);
    }
    if (tid == 0) *scale = now;
}

template <int D>
ER_DEV void kv8_append(const ErAppendArgs &p) {
    __shared__ float peaks[4];
    if (blockIdx.x >= p.cacheBlocks)
        turn_query_row<D>(p);
    else if (p.c.shift == 4)
        append_block<D, 16>(p, peaks);
    else if (p.c.shift == 5)
        append_block<D, 32>(p, peaks);
    else
        append_block<D, 64>(p, peaks);
}

#define ER_KV8_KERNELS(D)                                                                                          \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS) er_qk_norm_rope_d##D(ErRopeArgs p) {              \
        qk_norm_rope<D>(p);                                                                                        \
    }                                                                                                              \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS) er_kv8_append_d##D(ErAppendArgs p) {              \
        kv8_append<D>(p);                                                                                          \
    }
ER_KV8_KERNELS(64)
ER_KV8_KERNELS(128)
ER_KV8_KERNELS(256)

#include "er_kv8_attn.hip"
