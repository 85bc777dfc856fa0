// er_choose.hip -- rules on logits and the choice (part of er_draft.hip).

// The order of candidates: the larger value, then the lower token.  NaN is
// never taken; ER_NO_TOKEN where nothing is left.
#define ER_NO_TOKEN 0xffffffffu
#define ER_NO_ROW 0xfffffffeu  // of a slice whose row belongs to no sequence
struct Candidate {
    float v;
    uint32_t token;
};
ER_DEV Candidate better(Candidate a, Candidate b) { return b.v > a.v || (b.v == a.v && b.token < a.token) ? b : a; }
template <int CTRL, int ROWS = 0xf>
ER_DEV Candidate dpp_better(Candidate a) {
    const int v = __float_as_int(a.v);
    Candidate b;
    b.v = __int_as_float(__builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xf, false));
    b.token = (uint32_t)__builtin_amdgcn_update_dpp((int)a.token, (int)a.token, CTRL, ROWS, 0xf, false);
    return better(a, b);
}
// The best of the wave's, in lane 63.
ER_DEV Candidate wave_best(Candidate a) {
    a = dpp_better<ER_DPP_QUAD_XOR1>(a);
    a = dpp_better<ER_DPP_QUAD_XOR2>(a);
    a = dpp_better<ER_DPP_ROW_HALF_MIRROR>(a);
    a = dpp_better<ER_DPP_ROW_MIRROR>(a);
    a = dpp_better<ER_DPP_ROW_BCAST15, 0xa>(a);
    return dpp_better<ER_DPP_ROW_BCAST31, 0xc>(a);
}

// What the rules know of a row's sequence, and the row's place in it.
struct LogitRow {
    uint32_t s;
    int row0, n;
    float repetition, presence, frequency;
    uint32_t known, entries;  // of the history and the biases
};
// Of sequence s, which may differ between lanes.  Nothing waits for anything else.
ER_DEV LogitRow logit_sequence(const ErChooseArgs &p, uint32_t s) {
    LogitRow r = {s, (int)s, 1, 1.0f, 0.0f, 0.0f, 0, 0};
    if (p.start) {
        const int rows = (int)p.rows;
        r.row0 = min(max(p.start[s], 0), rows);
        r.n = min(max(min(p.start[s + 1], rows) - r.row0, 0), (int)p.maxRows);
    }
    if (p.penalty) {
        const float *w = p.penalty + 3 * (size_t)s;
        r.repetition = w[0], r.presence = w[1], r.frequency = w[2];
        if (p.history) r.known = min((uint32_t)max(p.historyLen[s], 0), p.historyStride);
    }
    if (p.bias) r.entries = min((uint32_t)max(p.biasLen[s], 0), p.biasStride);
    return r;
}
// Lanes look at a sequence each; false: the row belongs to none.
ER_DEV bool logit_row(const ErChooseArgs &p, uint32_t row, uint32_t lane, LogitRow &r) {
    if (!p.start) {
        if (row >= p.sequences) return false;
        r = logit_sequence(p, row);
        return true;
    }
    for (uint32_t at = 0; at < p.sequences; at += 64) {
        const LogitRow l = logit_sequence(p, min(at + lane, p.sequences - 1));
        const uint64_t has = __ballot((int)row >= l.row0 && (int)row < l.row0 + l.n);
        if (!has) continue;
        const uint32_t i = (uint32_t)__ffsll((unsigned long long)has) - 1u;
        r = LogitRow{lane_of(l.s, i), (int)lane_of((uint32_t)l.row0, i), (int)lane_of((uint32_t)l.n, i),
                     scalar_of(l.repetition, i), scalar_of(l.presence, i), scalar_of(l.frequency, i),
                     lane_of(l.known, i), lane_of(l.entries, i)};
        return true;
    }
    return false;
}

// The largest of the wave's, none of which is NaN, in lane 63.
template <int CTRL, int ROWS = 0xf>
ER_DEV float dpp_most(float a) {
    const int v = __float_as_int(a);
    const float b = __int_as_float(__builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xf, false));
    return b > a ? b : a;
}
ER_DEV float wave_most(float a) {
    a = dpp_most<ER_DPP_QUAD_XOR1>(a);
    a = dpp_most<ER_DPP_QUAD_XOR2>(a);
    a = dpp_most<ER_DPP_ROW_HALF_MIRROR>(a);
    a = dpp_most<ER_DPP_ROW_MIRROR>(a);
    a = dpp_most<ER_DPP_ROW_BCAST15, 0xa>(a);
    return dpp_most<ER_DPP_ROW_BCAST31, 0xc>(a);
}

// Four of a row's or list's n values from i on, which is a multiple of 4: read without
// a branch, that the loads of many be in flight at once, from the last four where the
// end lies among them or before; four_of then moves them into their places.  FOUR: n is
// 4 or more.  Else a branch on that, whose loads may not have been issued, costs exact
// waits for what was loaded before.
template <bool FOUR, typename T>
ER_DEV u32x4 load_four(const T *list, uint32_t i, uint32_t n) {
    if (FOUR || n >= 4) return *(const u32x4_a4 *)(list + min(i, n - 4));  // of one answer for all lanes
    const uint32_t *w = (const uint32_t *)list;
    u32x4 r = {0, 0, 0, 0};
    if (n > 0) r.x = w[0];
    if (n > 1) r.y = w[1];
    if (n > 2) r.z = w[2];
    return r;
}
ER_DEV u32x4 four_of(u32x4 r, uint32_t i, uint32_t n) {
    if (n >= 4 && i < n && i + 4 > n) {
        const uint32_t past = i + 4 - n;
        r = past == 1 ? u32x4{r.y, r.z, r.w, 0} : past == 2 ? u32x4{r.z, r.w, 0, 0} : u32x4{r.w, 0, 0, 0};
    }
    return r;
}

// One slice of one row: S times four logits of a thread (S > 1: the vocabulary has a
// slice at least), on their way while LDS takes what the rules say.  There how often
// the context has each token of the slice is counted, whole numbers whose order does not
// matter, and so is which entry of the biases is a token's last.  Tokens that any rule
// changes, a few of a hundred, are listed and then worked through side by side: formed
// in 64 bits and rounded once, each in the place of its count.
//
// Reads and writes the logits once, which bounds it: 172 nodes of 128256 logits, 4/32
// bytes of masks each, 41.7 us with the join, 4.2 TB/s.  64 rows with 4096 tokens of
// context and biases take 22.7 us, 2.9 TB/s, without them 14.9: the more of a workgroup's
// time passes between its reads and its writes, the fewer bytes are under way.  Counts
// that answer (to list a token when it is first met) took 25.1, with a lane's dummy for
// tokens of other slices, so that no branch lies between them, 26.5.  The rules in 64 bits
// in place, by whoever holds the logit, 33.
template <int S>
ER_DEV void choose_slice(const ErChooseArgs &p, uint32_t *lds) {
    constexpr uint32_t STEP = 4 * ER_CHOOSE_THREADS, SLICE = S * STEP, NONE = 0xffffffffu, WAVES = ER_CHOOSE_THREADS / 64;
    const uint32_t row = blockIdx.x / p.slices, at = blockIdx.x % p.slices, tid = threadIdx.x, lane = tid & 63u;
    const uint32_t from = at * SLICE, n = min(p.vocab - from, SLICE);
    LogitRow r;
    if (!logit_row(p, row, lane, r)) {
        if (p.chosen && p.slices > 1 && tid == 0) p.partI[blockIdx.x] = ER_NO_ROW;
        return;
    }
    const bool counts = !(r.repetition == 1.0f && r.presence == 0.0f && r.frequency == 0.0f);
    const double repetition = r.repetition, presence = r.presence, frequency = r.frequency;
    const uint32_t known = counts ? r.known : 0, drafts = counts && p.seen ? (uint32_t)r.n : 0, entries = r.entries;
    const int32_t *history = p.history + (size_t)r.s * p.historyStride;
    // Loads return in order: those that LDS waits for come first.
    uint32_t words[S];
#pragma unroll
    for (int j = 0; j < S; ++j) words[j] = ~0u;
    if (p.allowed) {
        const uint32_t *w = p.allowed + (size_t)row * p.allowedStride;
#pragma unroll
        for (int j = 0; j < S; ++j) words[j] = w[(from + min(j * STEP + 4 * tid, n - 1)) >> 5];
    }
    u32x4 past[4] = {};
    if (known) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) past[j] = load_four<false>(history, 4 * tid + j * STEP, known);
    }
    const int32_t *biased = p.biasToken + (size_t)r.s * p.biasStride;
    uint32_t first = ER_NO_TOKEN;  // this thread's first entry of the biases
    if (entries) first = (uint32_t)biased[min(tid, entries - 1)];
    const float *x = p.logits + (size_t)row * p.stride;
    u32x4 raw[S];
#pragma unroll
    for (int j = 0; j < S; ++j) raw[j] = load_four<(S > 1)>(x, from + j * STEP + 4 * tid, p.vocab);
    bool changed = false;
    if (known + drafts + entries > 0) {
        // NONE + how often the context has the token, then the bits of its value; a
        // value whose bits are NONE is another NaN.
        uint32_t *times = lds, *entry = lds + SLICE;
        uint16_t *list = (uint16_t *)(entry + (p.bias ? SLICE : 0));
        __shared__ uint32_t listed;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const uint32_t i = j * STEP + 4 * tid;
            *(u32x4 *)(times + i) = u32x4{NONE, NONE, NONE, NONE};
            if (entries) *(u32x4 *)(entry + i) = u32x4{0, 0, 0, 0};
        }
        if (tid == 0) listed = 0;
        __syncthreads();
        // Few of the context's tokens lie in the slice, and no lane asks for an answer.
        auto count = [&](uint32_t t) {
            if (t < n) atomicAdd(times + t, 1u);
        };
        auto count_past = [&](uint32_t base) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                if (base + j * STEP >= known) break;  // of one answer for all lanes
                const uint32_t i = base + j * STEP + 4 * tid;
                const u32x4 t = four_of(past[j], i, known);
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) count(i + k < known ? t[k] - from : NONE);
            }
        };
        count_past(0);
        for (uint32_t base = 4 * STEP; base < known; base += 4 * STEP) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) past[j] = load_four<false>(history, base + j * STEP + 4 * tid, known);
            count_past(base);
        }
        for (uint32_t i = tid; i < drafts; i += ER_CHOOSE_THREADS) {
            const uint32_t word = p.seen[(size_t)row * p.words + (i >> 5)], token = (uint32_t)p.token[r.row0 + i];
            count(word >> (i & 31u) & 1u ? token - from : NONE);
        }
        for (uint32_t i = tid; i < entries; i += ER_CHOOSE_THREADS) {
            const uint32_t t = (i == tid ? first : (uint32_t)biased[i]) - from;
            if (t < n) atomicMax(entry + t, i + 1);
        }
        __syncthreads();
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const uint32_t i = j * STEP + 4 * tid;
            const u32x4 w = *(const u32x4 *)(times + i);
            const u32x4 e = entries ? *(const u32x4 *)(entry + i) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 4; ++k) mine |= (w[k] + 1) | e[k] ? 1u << (4 * j + k) : 0u;
        }
        if (mine) {
            uint32_t to = atomicAdd(&listed, (uint32_t)__popc(mine));
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (mine >> (4 * j + k) & 1u) list[to++] = (uint16_t)(j * STEP + 4 * tid + k);
        }
        __syncthreads();
        const uint32_t all = uniform(listed);
        changed = all != 0;
        if (changed) {
            for (uint32_t i = tid; i < all; i += ER_CHOOSE_THREADS) {
                const uint32_t t = list[i], c = times[t] + 1, e = entries ? entry[t] : 0u;
                double d = (double)x[from + t];
                if (c) d = (d > 0.0 ? d / repetition : d * repetition) - (presence + frequency * (double)c);
                if (e) d += (double)p.bias[(size_t)r.s * p.biasStride + e - 1];
                const float f = (float)d;
                times[t] = f == f ? __float_as_uint(f) : 0x7fc00000u;
            }
            __syncthreads();
        }
    }
    float *y = p.out ? p.out + (size_t)row * p.stride + from : nullptr;
    float most = -__builtin_inff();
    f32x4 v[S];
    uint32_t bits[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const uint32_t i = j * STEP + 4 * tid;
        u32x4 u = four_of(raw[j], from + i, p.vocab);
        if (changed) {
            const u32x4 w = *(const u32x4 *)(lds + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = w[k] == NONE ? u[k] : w[k];
        }
        bits[j] = words[j] >> (i & 31u) & (i + 4 <= n ? 15u : i < n ? 15u >> (i + 4 - n) : 0u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[j][k] = bits[j] >> k & 1u ? __uint_as_float(u[k]) : -__builtin_inff();
            most = v[j][k] > most ? v[j][k] : most;
        }
        if (y) {
            if (i + 4 <= n) {
                __builtin_nontemporal_store(v[j], (f32x4_a4 *)(y + i));
            } else {
                if (i < n) y[i] = v[j].x;
                if (i + 1 < n) y[i + 1] = v[j].y;
                if (i + 2 < n) y[i + 2] = v[j].z;
            }
        }
    }
    if (!p.chosen) return;
    // The largest first, then the lowest of the allowed tokens that have it.
    __shared__ float waves[WAVES];
    __shared__ uint32_t token;
    const float whole = wave_most(most);
    if (lane == 63) waves[tid >> 6] = whole;
    if (tid == 0) token = ER_NO_TOKEN;
    __syncthreads();
    float top = waves[0];
#pragma unroll
    for (uint32_t i = 1; i < WAVES; ++i) top = waves[i] > top ? waves[i] : top;
    if (most == top) {
        uint32_t mine = ER_NO_TOKEN;
#pragma unroll
        for (int j = S - 1; j >= 0; --j)
#pragma unroll
            for (int k = 3; k >= 0; --k)
                if ((bits[j] >> k & 1u) && v[j][k] == top) mine = from + j * STEP + 4 * tid + k;
        if (mine != ER_NO_TOKEN) atomicMin(&token, mine);
    }
    __syncthreads();
    if (tid == 0) {
        if (p.slices == 1) {
            p.chosen[row] = (int)token;
        } else {
            p.partV[blockIdx.x] = top;
            p.partI[blockIdx.x] = token;
        }
    }
}

extern __shared__ __attribute__((aligned(16))) uint32_t er_choose_lds[];
#define ER_CHOOSE(S) \
    extern "C" __global__ void __launch_bounds__(ER_CHOOSE_THREADS) er_choose_s##S(ErChooseArgs p) { choose_slice<S>(p, er_choose_lds); }
ER_CHOOSE(1)
ER_CHOOSE(2)

// The best of a row's slices: a wave a row.  What it needs to know of the row stands in
// its slices, so that it waits for memory once.
extern "C" __global__ void __launch_bounds__(ER_CHOOSE_THREADS) er_choose_join(ErChooseArgs p) {
    const uint32_t row = uniform((blockIdx.x * ER_CHOOSE_THREADS + threadIdx.x) >> 6), lane = threadIdx.x & 63u;
    if (row >= p.rows) return;
    Candidate best = {-__builtin_inff(), ER_NO_TOKEN};
    bool none = false;
    for (uint32_t i = lane; i < p.slices; i += 64) {
        const Candidate c = {p.partV[(size_t)row * p.slices + i], p.partI[(size_t)row * p.slices + i]};
        none = c.token == ER_NO_ROW;
        best = better(best, c);
    }
    if (__ballot(none)) return;
    best = wave_best(best);
    if (lane == 63) p.chosen[row] = (int)best.token;
}
