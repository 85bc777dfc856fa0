// er_kv8_few.hip -- attention under masks for few columns: decode, trees of
// drafts, short chunks (part of er_draft.hip).
//
// The narrow kernel's tiles and products, for NB blocks of 16 columns a wave: a
// tile's codes are converted once for all of them.  Like the narrow kernel's,
// units (sequence, head, 16 NB columns) lie on one line that the resident
// workgroups share evenly; a workgroup's four waves take its tiles in turn.
//
// Decode is bound by memory: 48 users of 32 over 8 heads of 128 read 777 MB in 140
// us, 5.5 TB/s.  Trees are bound by issue: those of 32 users (639 rows of 32 heads over
// 8 of 128, fp32) take 143 us with the join, of which vector instructions
// are 59% of the SIMDs' cycles and products 32%; a tile costs a SIMD some 1325 cycles
// with one block of columns.  One user's call is a chain of loads, 8 to 10 us.

#define ER_DEV_MEMBER __device__ __forceinline__

// Units of a sequence and key/value head.
template <int NB>
ER_DEV uint32_t few_blocks(const ErAttendArgs &p, const Sequence &q) {
    return ((uint32_t)q.n * p.group + (16u * NB - 1)) / (16u * NB);
}
ER_DEV uint32_t few_length(uint32_t steps, bool aligned, uint32_t quota) {
    return aligned ? (steps + quota - 1) / quota * quota : steps;
}
// Shares of ER_FEW_LEAST steps (half of it where half the workgroups do) and, as long
// as the units do not fit the workgroups so, half as many again: a workgroup that
// takes two units starts and ends twice.  Past four times that it counts less than an
// even share.  16 draft checks at head width 256, 64 units of up to 47 steps: 25 us by
// 6 steps, 31 by 4 across units.  By 2, 3, 4, 6 steps, us: a user of 8000 tokens 18.3,
// 17.0, 14.0, 15.7; where 2 leave half the workgroups without work, one user's tree of
// 26 drafts 13.7, 13.7, 14.6, 15.0, a window of 1020 tokens 12.4, 12.9, 12.8, 13.5.
constexpr uint32_t few_next(uint32_t quota) { return quota < ER_FEW_LEAST ? ER_FEW_LEAST : quota + quota / 2; }
template <int NB, uint32_t QUOTA, class A>
ER_DEV Shares few_shares_by(const A &p, const LaneSequence &first, uint32_t lane) {
    Shares s;
    s.aligned = QUOTA <= 4 * ER_FEW_LEAST;
    s.quota = s.aligned ? QUOTA : 1;
    uint32_t sum = 0;
    for (uint32_t at = 0; at < p.b.sequences; at += 64) {
        const LaneSequence l = at ? lane_sequence(p, at + lane) : first;
        sum += few_length(l.steps, s.aligned, s.quota) * few_blocks<NB>(p, l.q);
    }
    s.total = wave_sum(sum) * p.c.heads;
    if constexpr (QUOTA > 4 * ER_FEW_LEAST) {
        s.quota = max(ER_FEW_LEAST, (s.total + p.shares - 1) / p.shares);
        return s;
    } else {
        if (s.total <= p.shares * (QUOTA < ER_FEW_LEAST ? QUOTA / 2 : QUOTA)) return s;
        return few_shares_by<NB, few_next(QUOTA)>(p, first, lane);
    }
}
template <int NB, class A>
ER_DEV Shares few_shares(const A &p, const LaneSequence &first, uint32_t lane) {
    return few_shares_by<NB, ER_FEW_LEAST / 2>(p, first, lane);
}
// The sequence that place `at` of the line belongs to, and where it begins.
template <int NB, class A>
ER_DEV uint32_t few_sequence_at(const A &p, const LaneSequence &first, const Shares &sh, uint32_t at, uint32_t lane,
                                uint32_t &begins) {
    uint32_t before = 0;
    for (uint32_t s0 = 0;; s0 += 64) {
        const LaneSequence l = s0 ? lane_sequence(p, s0 + lane) : first;
        const uint32_t mine = few_length(l.steps, sh.aligned, sh.quota) * few_blocks<NB>(p, l.q) * p.c.heads, upTo = wave_prefix(mine);
        const uint64_t past = __ballot(before + upTo > at);
        if (past || s0 + 64 >= p.b.sequences) {
            const uint32_t i = past ? (uint32_t)__ffsll((unsigned long long)past) - 1u : 63u;
            begins = before + lane_of(upTo - mine, i);
            return s0 + i;
        }
        before += lane_of(upTo, 63);
    }
}

// Running state of a wave's columns: n, 16 + n, ...
template <int D, int NB>
struct FewState {
    f32x4 o[NB * (D / 16)];  // as NarrowState's, one block's behind the other's
    float m[NB], l[NB], vref, vinv;
    // Bits 4 b .. 4 b + 3 and 16 further on: block b's columns saw a token; bit 31:
    // a masked tile held NaN codes.  Not truth values, some of which the compiler
    // lost where it kept them as masks of lanes through a loop.
    uint32_t flags;
};

// As attend_narrow, with `masked` the same for the wave.
template <int D, int NB, int TERMS, class A>
ER_DEV void attend_few(FewState<D, NB> &st, NarrowTile<D> &t, const h8 (&qb)[NB][TERMS][D / 32], const float (&qf)[NB], const A &p,
                       int T, const uint32_t (&shown32)[NB], bool masked, const Spans &w, uint32_t g, float &vtop) {
    constexpr int J = D / 16;
    const bool ok0 = t.page[0] >= 0, ok1 = t.page[1] >= 0;
    f32x4 s[NB][2] = {};
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const u32x4 c = t.k[half][k / 2];
            const h8 a = k % 2 ? codes_to_h8(c.z, c.w) : codes_to_h8(c.x, c.y);
#pragma unroll
            for (int term = 0; term < TERMS; ++term)
#pragma unroll
                for (int b = 0; b < NB; ++b) s[b][half] = mfma16(a, qb[b][term][k], s[b][half]);
        }
    if (masked) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int tok = T + 16 * (i / 4) + 4 * (int)g + (i & 3);
            const bool ok = i < 4 ? ok0 : ok1;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                s[b][i / 4][i & 3] = ok && (shown32[b] >> (16 * (i / 4) + (i & 3)) & 1u) ? s[b][i / 4][i & 3] : -__builtin_inff();
#pragma unroll
            for (int d = 0; d < D / 64; ++d) {
                const uint32_t v = ok && touches(p, tok, tok + 1, w.anyLo, w.anyHi) ? t.v[d][i] : 0u, nan = nan_codes(v);
                st.flags |= nan ? 1u << 31 : 0u;
                t.v[d][i] = v & ~nan;
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) st.flags |= (shown32[b] & ((ok0 ? 0xfu : 0u) | (ok1 ? 0xf0000u : 0u))) << 4 * b;
    const float ks0 = ok0 ? t.ks[0] : t.ks[1], ks1 = ok1 ? t.ks[1] : t.ks[0];
    float f0[NB], f1[NB];
    bool above = false;
    float top[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        f0[b] = score_factor(qf[b], ks0);
        f1[b] = score_factor(qf[b], ks1);
        top[b] = fmaxf(fmaxf(fmaxf(s[b][0].x, s[b][0].y), fmaxf(s[b][0].z, s[b][0].w)) * f0[b],
                       fmaxf(fmaxf(s[b][1].x, s[b][1].y), fmaxf(s[b][1].z, s[b][1].w)) * f1[b]);
        above |= top[b] - st.m[b] > ER_ROOM;
    }
    if (__any(above)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float to = fmaxf(st.m[b], reference_of(column_max4(top[b]))), f = __builtin_amdgcn_exp2f(st.m[b] - to);
            st.m[b] = to;
            st.l[b] *= f;
#pragma unroll
            for (int j = 0; j < J; ++j) st.o[b * J + j] *= f;
        }
    }
    const float vs0 = ok0 ? t.vs[0] : t.vs[1], vs1 = ok1 ? t.vs[1] : t.vs[0];
    ScaleRange r = {0u, ~0u};
    r.add(__float_as_uint(uniform(vs0)));
    r.add(__float_as_uint(uniform(vs1)));
    follow_scale(r, vtop, st.vref, st.vinv, st.o);
    h8 weights[NB][TERMS];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(s[b][i / 4][i & 3] * (i < 4 ? f0[b] : f1[b]) - st.m[b]);
        st.l[b] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        weight_terms<TERMS>(x, weights[b]);
    }
    const float v0 = vs0 * st.vinv, v1 = vs1 * st.vinv;
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
        h8 a[4];
        transpose_codes(t.v[d], v0, v1, a);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int term = 0; term < TERMS; ++term)
#pragma unroll
                for (int b = 0; b < NB; ++b) st.o[b * J + 4 * d + j] = mfma16(a[j], weights[b][term], st.o[b * J + 4 * d + j]);
    }
}

// load_query, its loads apart from its conversions, for columns that are there.
template <int N>
ER_DEV void query_values(const float *src, float (&x)[N][8]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float *v = src + k / 2 * 64 + k % 2 * 8;
        const f32x4 lo = *(const f32x4_a4 *)v, hi = *(const f32x4_a4 *)(v + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[k][i] = lo[i];
            x[k][4 + i] = hi[i];
        }
    }
}
template <int N, int TERMS>
ER_DEV float query_terms(float (&x)[N][8], float scale, h8 (&b)[TERMS][N]) {
    float peak = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[k][i] *= scale;
            peak = fmaxf(peak, finite_magnitude(x[k][i]));
        }
    peak = column_max4(peak);
    const int e = min(max((int)(__float_as_uint(peak) >> 23) - 126, -126), 126);
    const float f = exp2i(-e);
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = x[k][i] * f;
            const _Float16 t = (_Float16)v;
            b[0][k][i] = t;
            if constexpr (TERMS == 2) b[1][k][i] = (_Float16)(v - (float)t);
        }
    return exp2i(e);
}

ER_DEV float scalar_of(float v, uint32_t lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// A tile's codes, as load_narrow brings them, from its halves' pages.
template <int D, int P>
ER_DEV void load_codes(NarrowTile<D> &t, const ErKv8Cache &c, uint32_t h, int T, uint32_t n, uint32_t g) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const size_t block = (size_t)(uint32_t)max(t.page[half], 0) * c.heads + h;
        const size_t base = block * (P * D) + ((uint32_t)(T + 16 * half) % P) * D;
        const uint8_t *kp = c.k + base + (n * D + 16 * g);
        const uint8_t *vp = c.v + base + (4 * g * D + n * (D / 16));
#pragma unroll
        for (int j = 0; j < D / 64; ++j) t.k[half][j] = *(const u32x4 *)(kp + 64 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            typedef uint32_t dwords __attribute__((ext_vector_type(D / 64 > 1 ? D / 64 : 2)));
            if constexpr (D == 64) {
                t.v[0][4 * half + i] = *(const uint32_t *)(vp + i * D);
            } else {
                const dwords x = *(const dwords *)(vp + i * D);
#pragma unroll
                for (int d = 0; d < D / 64; ++d) t.v[d][4 * half + i] = x[d];
            }
        }
    }
}

// Columns [col0, col0 + cols) of one unit against steps [from, to) of its
// tokens; otherwise as narrow_unit.
template <int D, int P, int NB, int TERMS, class A>
ER_DEV void few_unit(const A &p, uint32_t s, const Sequence &q, uint32_t h, uint32_t col0, uint32_t cols, uint32_t from,
                     uint32_t to, bool complete, uint32_t part, float *lds, uint32_t (*drafts)[ER_DRAFT_WORDS]) {
    constexpr int J = D / 16;
    constexpr bool TWO = D < 256;  // two tiles in registers
    constexpr uint32_t WIDE = 16 * NB;
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const uint32_t lane = tid & 63u, wave = uniform(tid >> 6), n = lane & 15u, g = lane >> 4;
    const Spans w = spans_of(p, q, col0, col0 + cols - 1);
    const Reach reach = reach_of(p, spans_of(p, q, 0, (uint32_t)q.n * p.group - 1));  // the steps are those of all columns
    const int begin = 64 * (int)from, end = min(w.anyHi - reach.skip, 64 * (int)to);
    auto column = [&](int b) { return column_of(p, q, h, col0 + min(16 * b + n, cols - 1)); };
    // The wave's tiles 64 (of pages of 16 tokens 32) at a time: lane i finds the page
    // and scales of the i-th (of half i % 2 of the i / 2-th), and which tiles there
    // are, and which all columns see whole, are bits of scalars.  (Read tile by tile
    // into scalars, the next tile's scales had to arrive before the present one's
    // could be used: scalar loads return out of order, so that every wait is one for
    // all.)  Where the halves of a tile that is not whole have value scales far apart,
    // it is taken half by half, as a column may see the small one alone.
    constexpr int PARTS = P < 32 ? 2 : 1, TOKENS = 32 / PARTS;
    constexpr uint64_t EACH = PARTS == 2 ? 0x5555555555555555ull : ~0ull;  // the bits that stand for tiles
    int from64 = begin + 32 * (int)wave, page = -1;
    float ks = 0.0f, vs = 0.0f;
    uint64_t wholes = 0, tiles = 0, halves = 0, seconds = 0;
    auto look = [&]() {
        const int x = from64 + 128 * (int)(lane / PARTS), mine = token_of(reach, x) + TOKENS * (int)(lane % PARTS);
        // not conditional, so that no branch waits for it
        const int k = page_of(p.b, p.c, s, min(mine, q.len - 1));
        page = x < end && touches(p, mine, mine + TOKENS, w.anyLo, w.anyHi) ? k : -1;
        const size_t block = (size_t)(uint32_t)max(page, 0) * p.c.heads + h;
        ks = p.c.ks[block];
        vs = p.c.vs[block];
        const uint64_t there = __ballot(page >= 0), whole = __ballot(page >= 0 && within(p, mine, mine + TOKENS, w.allLo, w.allHi));
        if constexpr (PARTS == 2) {
            wholes = whole & whole >> 1 & EACH;
            tiles = (there | there >> 1) & EACH;
            ScaleRange r = {0u, ~0u};
            r.add(__float_as_uint(vs));
            r.add((uint32_t)__builtin_amdgcn_update_dpp(0, __float_as_int(vs), ER_DPP_QUAD_XOR1, 0xf, 0xf, false));
            halves = seconds = __ballot(r.apart()) & there & there >> 1 & EACH & ~wholes;
        } else {
            wholes = whole;
            tiles = there;
        }
    };
    struct Next {
        uint32_t i;
        bool masked;
    };
    auto load = [&](NarrowTile<D> &t) {
        const bool second = PARTS == 2 && tiles == 0;
        const uint64_t bits = second ? seconds : tiles;
        const uint32_t i = bits ? (uint32_t)__builtin_ctzll(bits) : 64u - PARTS, j = i + PARTS - 1;
        t.page[0] = __builtin_amdgcn_readlane(page, i);
        t.page[1] = __builtin_amdgcn_readlane(page, j);
        if (PARTS == 2 && second) {
            t.page[0] = -1;
            seconds &= seconds - 1;
        } else {
            if (PARTS == 2 && halves >> i & 1u) t.page[1] = -1;
            tiles &= tiles - 1;
        }
        t.ks[0] = scalar_of(ks, i);
        t.vs[0] = scalar_of(vs, i);
        t.ks[1] = scalar_of(ks, j);
        t.vs[1] = scalar_of(vs, j);
        load_codes<D, P>(t, p.c, h, token_of(reach, from64 + 128 * (int)(i / PARTS)), n, g);
        return Next{i, !(wholes >> i & 1u)};
    };
    // The first tile is on its way before the query is read: its pages are the
    // longest chain of loads.
    NarrowTile<D> t0, t1;
    Next n0 = {63u, false}, n1;
    int left = 0;
    if (from64 < end) {
        look();
        left = __builtin_popcountll(tiles) + __builtin_popcountll(seconds);
        n0 = load(t0);
    }
    // All of a query's loads before its conversions; of columns that are not there
    // the last one's, which no one reads.
    h8 qb[NB][TERMS][D / 32];
    float qf[NB], values[NB][D / 32][8];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const Column c = column(b);
        query_values(p.q + (size_t)c.row * p.qStride + (size_t)c.head * D + 16 * g, values[b]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) qf[b] = query_terms(values[b], p.scale, qb[b]);
    // The drafts' bits, as in the wide kernel.
    int draftsFrom = 0x7fffffff;
    if (p.seen && token_of(reach, max(min(w.anyHi - reach.skip, 64 * (int)to) - 1, 0)) >= w.allHi) {
        draftsFrom = w.allHi & ~31;
        const int words = (((w.anyHi + 63) & ~63) - draftsFrom) >> 5;
        for (int i = (int)tid; i < (int)WIDE * words; i += ER_KV8_THREADS) {
            const uint32_t col = (uint32_t)(i / words);
            const int word = i - (int)col * words;
            drafts[col][word] = drafts_at(p, q, column_of(p, q, h, col0 + min(col, cols - 1)), draftsFrom + 32 * word);
        }
        __syncthreads();
    }
    FewState<D, NB> st = {};
    float vtop = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b) st.m[b] = ER_NO_MAX;
    auto attend = [&](NarrowTile<D> &t, const Next &at) {
        uint32_t shown[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) shown[b] = ~0u;
        const int token = token_of(reach, from64 + 128 * (int)(at.i / PARTS));
        if (at.masked) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                shown[b] = sees32(p, column(b), token);
                if (token >= draftsFrom) shown[b] |= drafts[16 * b + n][(token - draftsFrom) >> 5];
                shown[b] >>= 4 * g;
            }
        }
        attend_few<D, NB, TERMS>(st, t, qb, qf, p, token, shown, at.masked, w, g, vtop);
    };
    // Two tiles are in registers at a time; loads are not conditional (behind the
    // last tile the first page is read once more), since a load that may not have
    // been issued makes every wait one for all loads.
    while (true) {
        if (left > 0) {
            if constexpr (TWO) {
                while (true) {
                    n1 = load(t1);
                    attend(t0, n0);
                    if (--left == 0) break;
                    n0 = load(t0);
                    attend(t1, n1);
                    if (--left == 0) break;
                }
            } else {
                while (true) {
                    attend(t0, n0);
                    if (--left == 0) break;
                    n0 = load(t0);
                }
            }
        }
        from64 += 64 / PARTS * 128;
        if (from64 >= end) break;
        look();
        left = __builtin_popcountll(tiles) + __builtin_popcountll(seconds);
        n0 = load(t0);
    }
    if (__any(st.flags >> 31)) {
        // each wave marks its own sums, for the tokens of all waves of its columns
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const Column c = column(b);
            for (int x = begin; x < end; ++x) {
                const int tok = token_of(reach, x);
                if (!(sees(p, c, tok) || (drafts_at(p, q, c, tok) & 1u))) continue;
                const int page = page_of(p.b, p.c, s, tok);
                if (page < 0) continue;
                const size_t slot = (((size_t)page * p.c.heads + h) << p.c.shift) + ((uint32_t)tok & ((1u << p.c.shift) - 1u));
                const uint8_t *v = p.c.v + slot * D;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < D / 64; ++d) {
                        const uint32_t nan = nan_codes(*(const uint32_t *)(v + (4 * g + i) * J + 4 * d));
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            st.o[b * J + 4 * d + j][i] = (nan >> (8 * j)) & 1u ? __builtin_nanf("") : st.o[b * J + 4 * d + j][i];
                    }
            }
        }
    }

    // the waves' columns, [wave][16 NB][D + 4], and their references and sums (-1: nothing seen)
    constexpr uint32_t PITCH = D + 4;
    constexpr uint32_t SLOTS = 4 * WIDE;
    float *sm = lds + SLOTS * PITCH, *sl = sm + SLOTS;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const uint32_t slot = wave * WIDE + 16 * b + n;
        const float l = column_sum4(st.l[b]);
        const bool seen = column_max4(st.flags & (0xf000fu << 4 * b) ? 1.0f : 0.0f) > 0.0f;
        float *at = lds + slot * PITCH;
        const float f = st.vref * 0.0078125f * over(l);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < J; j += 4)
                *(f32x4 *)(at + (4 * g + i) * J + j) = f32x4{st.o[b * J + j][i] * f, st.o[b * J + j + 1][i] * f,
                                                            st.o[b * J + j + 2][i] * f, st.o[b * J + j + 3][i] * f};
        if (g == 0) {
            sm[slot] = st.m[b];
            sl[slot] = seen ? l : -1.0f;
        }
    }
    __syncthreads();
    const uint32_t d = (tid % (D / 4)) * 4;
#pragma unroll 1
    for (uint32_t col = tid / (D / 4); col < cols; col += ER_KV8_THREADS / (D / 4)) {
        float m[4], l[4], top = ER_NO_MAX, total = 0.0f;
        f32x4 v[4], o = {};
        bool visible = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = sm[col + WIDE * i];
            l[i] = sl[col + WIDE * i];
            v[i] = *(const f32x4 *)(lds + (col + WIDE * i) * PITCH + d);
            top = fmaxf(top, m[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            visible |= !(l[i] < 0.0f);
            m[i] = l[i] < 0.0f ? 0.0f : l[i] * __builtin_amdgcn_exp2f(m[i] - top);
            total += m[i];
        }
        const float inverse = over(total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!(l[i] < 0.0f)) o += v[i] * (m[i] * inverse);
        if (complete) {
            const Column k = column_of(p, q, h, col0 + col);
            store4(p, k.row, k.head, d, D, joined(o, visible, total));
        } else {
            const size_t to = (size_t)part * WIDE + col;
            if (visible) *(f32x4 *)(p.partO + to * D + d) = o;
            if (d == 0) *(f32x2 *)(p.partML + 2 * to) = f32x2{top, visible ? total : -1.0f};
        }
    }
}

template <int D, int P, int NB, int TERMS, class A>
ER_DEV void kv8_attend_few(const A &p, float *lds, uint32_t (*drafts)[ER_DRAFT_WORDS]) {
    constexpr uint32_t WIDE = 16 * NB;
    const uint32_t H = p.c.heads, lane = threadIdx.x & 63u;
    // Without shares a workgroup has one unit (p.tiles a sequence and head).
    uint32_t s, unit, at, last, begins, length, place = blockIdx.x;
    Shares sh = {};
    LaneSequence l;
    if (p.shares == 0) {
        s = blockIdx.x / p.tiles / H;
        l = lane_sequence(p, s);
        const uint32_t block = blockIdx.x % p.tiles, blocks = few_blocks<NB>(p, l.q);
        if (block >= blocks) return;
        unit = blockIdx.x / p.tiles % H * blocks + block;
        at = begins = 0;
        last = length = l.steps;
    } else {
        const LaneSequence first = lane_sequence(p, lane);
        sh = few_shares<NB>(p, first, lane);
        // Workgroups go to the 8 XCDs in turn.  Where all have work, those of an XCD
        // take places that follow each other: units that read the same cache do too,
        // and one L2 then serves them.
        if (!sh.aligned && p.shares % 8 == 0) place = blockIdx.x % 8 * (p.shares / 8) + blockIdx.x / 8;
        at = place * sh.quota;
        last = min(at + sh.quota, sh.total);
        if (at >= last) return;
        s = few_sequence_at<NB>(p, first, sh, at, lane, begins);
        l = lane_sequence_at(p, first, s);
        // as in kv8_attend_narrow
        if (l.steps == 0) return;
        length = few_length(l.steps, sh.aligned, sh.quota);
        unit = (at - begins) / length;
        if (unit >= H * few_blocks<NB>(p, l.q)) return;
        begins += unit * length;
    }
    while (true) {
        const uint32_t blocks = few_blocks<NB>(p, l.q), from = at - begins, to = min(last - begins, l.steps);
        const uint32_t col0 = unit % blocks * WIDE, cols = min((uint32_t)l.q.n * p.group - col0, WIDE);
        if (from < to)  // else nothing but what rounds a unit's length up
            few_unit<D, P, NB, TERMS>(p, s, l.q, unit / blocks, col0, cols, from, to, from == 0 && to == l.steps,
                                      2 * place + (from == 0 ? 1u : 0u), lds, drafts);
        begins += length;
        at = begins;
        if (at >= last) return;
        if (++unit == H * blocks) {
            unit = 0;
            do {
                if (++s >= p.b.sequences) return;
                l = lane_sequence(p, s);
            } while (l.steps == 0);
            length = few_length(l.steps, sh.aligned, sh.quota);
        }
        __syncthreads();  // the sums in LDS have been read
    }
}

// Where a column's parts lie, once its row's sequence is known.
struct FewParts {
    uint32_t w0, parts;  // the first workgroup that had some of the unit's steps; how many did
    uint32_t slot, col;  // columns of a part, and the place of this one
    ER_DEV_MEMBER size_t index(uint32_t i) const {
        return (size_t)(2 * (w0 + i) + (i == 0 ? 1u : 0u)) * slot + col;
    }
};
// The line up to sequence s, which a row belongs to; all lanes take part.  False:
// the row belongs to none.
template <int NB, class A>
ER_DEV bool few_line(const A &p, uint32_t row, uint32_t lane, LaneSequence &l, Shares &sh, uint32_t &before) {
    const LaneSequence first = lane_sequence(p, lane);
    uint32_t s;
    if (p.b.sequences <= 64) {  // no second read of their starts
        const uint64_t has = __ballot((int)row >= first.q.row0 && (int)row < first.q.row0 + first.q.n);
        if (!has) return false;
        s = (uint32_t)__ffsll((unsigned long long)has) - 1u;
    } else {
        s = uniform(sequence_of_row(p.b, row, lane));
        if (s >= p.b.sequences) return false;
    }
    l = lane_sequence_at(p, first, s);
    if ((int)row < l.q.row0 || (int)row >= l.q.row0 + l.q.n) return false;
    sh = few_shares<NB>(p, first, lane);
    before = 0;
    for (uint32_t i = lane; i < s; i += 64) {
        const LaneSequence b = i < 64 ? first : lane_sequence(p, i);
        before += few_length(b.steps, sh.aligned, sh.quota) * few_blocks<NB>(p, b.q);
    }
    before = wave_sum(before) * p.c.heads;
    return true;
}
template <int NB, class A>
ER_DEV FewParts few_parts(const A &p, const LaneSequence &l, const Shares &sh, uint32_t before, uint32_t row, uint32_t head) {
    const uint32_t col = (row - (uint32_t)l.q.row0) * p.group + head % p.group;
    const uint32_t unit = head / p.group * few_blocks<NB>(p, l.q) + col / (16 * NB);
    const uint32_t begins = before + unit * few_length(l.steps, sh.aligned, sh.quota);
    FewParts r;
    r.w0 = begins / sh.quota;
    r.parts = (begins + l.steps - 1) / sh.quota - r.w0 + 1;
    r.slot = 16 * NB;
    r.col = col % (16 * NB);
    // one workgroup had it all and wrote it; or the arrays have changed, as in kv8_attend_narrow
    if (r.parts == 1 || r.w0 + r.parts > p.shares) r.parts = 0;
    return r;
}

// One column (a row of a query head) a workgroup: many parts of few columns, one
// user far into a document.  Up to 64 parts, a lane's references and sums and the first
// outputs are asked for at once.
template <int D, int NB, class A>
ER_DEV void few_join_column(const A &p, float *lds) {
    constexpr uint32_t LANES = D / 4, AT_ONCE = ER_KV8_THREADS / LANES, EARLY = 64 / AT_ONCE < 4 ? 64 / AT_ONCE : 4;
    const uint32_t heads = p.group * p.c.heads, row = blockIdx.x / heads, head = blockIdx.x % heads;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    LaneSequence l;
    Shares sh;
    uint32_t before;
    if (!few_line<NB>(p, row, lane, l, sh, before)) return;
    const FewParts f = few_parts<NB>(p, l, sh, before, row, head);
    if (f.parts == 0) return;
    if (f.parts > 64) {
        join_parts<D>(p, f.parts, (int)row, head, lds, [&](uint32_t i) { return f.index(i); });
        return;
    }
    const uint32_t mine = tid / LANES, d = (tid % LANES) * 4;
    const f32x2 ml = *(const f32x2 *)(p.partML + 2 * f.index(min(lane, f.parts - 1)));
    f32x4 early[EARLY];
#pragma unroll
    for (uint32_t k = 0; k < EARLY; ++k)
        early[k] = *(const f32x4 *)(p.partO + f.index(min(mine + k * AT_ONCE, f.parts - 1)) * D + d);
    const bool some = lane < f.parts && !(ml.y < 0.0f);
    const float top = wave_top(ml.x);
    float weight = some ? ml.y * __builtin_amdgcn_exp2f(ml.x - top) : 0.0f;
    // every wave has the sum, of the same terms in the same order
    const float total = group_sum<64>(weight);
    const bool seen = __any(some);
    weight = some ? share_of(weight, total) : -1.0f;
    f32x4 o = {};
#pragma unroll
    for (uint32_t k = 0; k < EARLY; ++k) {
        const uint32_t i = mine + k * AT_ONCE;
        const float w = __shfl(weight, (int)(i & 63u));
        if (i < f.parts && (w >= 0.0f || w != w)) o += early[k] * w;
    }
    for (uint32_t i0 = EARLY * AT_ONCE; i0 < f.parts; i0 += AT_ONCE) {
        const uint32_t i = i0 + mine;
        const float w = __shfl(weight, (int)(i & 63u));
        if (i < f.parts && (w >= 0.0f || w != w)) o += *(const f32x4 *)(p.partO + f.index(i) * D + d) * w;
    }
    *(f32x4 *)(lds + 4 * tid) = o;
    __syncthreads();
    if (tid < LANES) {
        f32x4 v = {};
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; ++k) v += *(const f32x4 *)(lds + 4 * (k * LANES + tid));
        store4(p, (int)row, head, 4 * tid, D, joined(v, seen, total));
    }
}

// D / 4 threads a column, whose parts, most often two or three, follow each
// other: 20448 columns of 32 trees took a workgroup each 46 us.
template <int D, int NB, class A>
ER_DEV void few_join(const A &p) {
    constexpr uint32_t AT_ONCE = ER_KV8_THREADS / (D / 4);
    const uint32_t heads = p.group * p.c.heads, strips = (heads + AT_ONCE - 1) / AT_ONCE;
    const uint32_t row = blockIdx.x / strips;
    const uint32_t head = blockIdx.x % strips * AT_ONCE + threadIdx.x / (D / 4), d = (threadIdx.x % (D / 4)) * 4;
    LaneSequence l;
    Shares sh;
    uint32_t before;
    if (!few_line<NB>(p, row, threadIdx.x & 63u, l, sh, before) || head >= heads) return;
    const FewParts f = few_parts<NB>(p, l, sh, before, row, head);
    if (f.parts == 0) return;
    float top = ER_NO_MAX, total = 0.0f;
    bool seen = false;
    f32x4 o = {};
    if (f.parts <= 4) {  // all that is read is asked for at once
        f32x2 ml[4];
        f32x4 part[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const size_t at = f.index(min(i, f.parts - 1));
            ml[i] = *(const f32x2 *)(p.partML + 2 * at);
            part[i] = *(const f32x4 *)(p.partO + at * D + d);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const bool some = i < f.parts && !(ml[i].y < 0.0f);
            ml[i].x = some ? ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - top) : 0.0f;
            seen |= some;
            total += ml[i].x;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (i < f.parts && !(ml[i].y < 0.0f)) o += part[i] * share_of(ml[i].x, total);
        store4(p, (int)row, head, d, D, joined(o, seen, total));
        return;
    }
    for (uint32_t i = 0; i < f.parts; ++i) top = fmaxf(top, p.partML[2 * f.index(i)]);
    for (uint32_t i = 0; i < f.parts; ++i) {
        const f32x2 ml = *(const f32x2 *)(p.partML + 2 * f.index(i));
        seen |= !(ml.y < 0.0f);
        total += ml.y < 0.0f ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - top);
    }
    for (uint32_t i = 0; i < f.parts; ++i) {
        const size_t at = f.index(i);
        const f32x2 ml = *(const f32x2 *)(p.partML + 2 * at);
        if (!(ml.y < 0.0f)) o += *(const f32x4 *)(p.partO + at * D + d) * share_of(ml.y * __builtin_amdgcn_exp2f(ml.x - top), total);
    }
    store4(p, (int)row, head, d, D, joined(o, seen, total));
}

#define ER_KV8_FEW(D, P, NB, TERMS, NAME, WAVES)                                                                   \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS, WAVES)                                            \
        er_kv8_masked_attend_c##NB##_d##D##_p##P##_##NAME(ErMaskedArgs p) {                                        \
        __shared__ __attribute__((aligned(16))) float sums[64 * NB * (D + 4) + 128 * NB];                          \
        __shared__ uint32_t drafts[16 * NB][ER_DRAFT_WORDS];                                                       \
        kv8_attend_few<D, P, NB, TERMS>(p, sums, drafts);                                                          \
    }
#define ER_KV8_FEWS(D, NB, TERMS, NAME, WAVES)                                                                     \
    ER_KV8_FEW(D, 16, NB, TERMS, NAME, WAVES)                                                                      \
    ER_KV8_FEW(D, 32, NB, TERMS, NAME, WAVES)                                                                      \
    ER_KV8_FEW(D, 64, NB, TERMS, NAME, WAVES)
ER_KV8_FEWS(64, 1, 1, bf16, 2)
ER_KV8_FEWS(64, 1, 2, f32, 2)
ER_KV8_FEWS(64, 2, 1, bf16, 2)
ER_KV8_FEWS(64, 2, 2, f32, 2)
ER_KV8_FEWS(128, 1, 1, bf16, 2)
ER_KV8_FEWS(128, 1, 2, f32, 2)
ER_KV8_FEWS(128, 2, 1, bf16, 2)
ER_KV8_FEWS(128, 2, 2, f32, 2)
ER_KV8_FEWS(256, 1, 1, bf16, 2)
// two pages a tile, two terms and wide heads need a few registers over the 256 that two waves leave
ER_KV8_FEW(256, 16, 1, 2, f32, 1)
ER_KV8_FEW(256, 32, 1, 2, f32, 2)
ER_KV8_FEW(256, 64, 1, 2, f32, 2)

#define ER_KV8_FEW_JOIN(D, NB)                                                                                     \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS) er_kv8_masked_join_c##NB##_d##D(ErMaskedArgs p) { \
        few_join<D, NB>(p);                                                                                        \
    }                                                                                                              \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS)                                                   \
        er_kv8_masked_join_column_c##NB##_d##D(ErMaskedArgs p) {                                                   \
        few_join_column<D, NB>(p, er_kv8_lds);                                                                     \
    }
ER_KV8_FEW_JOIN(64, 1)
ER_KV8_FEW_JOIN(64, 2)
ER_KV8_FEW_JOIN(128, 1)
ER_KV8_FEW_JOIN(128, 2)
ER_KV8_FEW_JOIN(256, 1)
