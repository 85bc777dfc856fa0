// er_choose.hip -- rules on logits and the choice (part of er_draft.hip).

// The order of candidates: the larger value, then the lower token.  NaN is
// never taken; ER_NO_TOKEN where nothing is left.
#define ER_NO_TOKEN 0xffffffffu
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

// The sequence of a row, and the row's place in it; false: it belongs to none.
struct LogitRow {
    uint32_t s;
    int row0, n;
};
ER_DEV bool logit_row(const ErChooseArgs &p, uint32_t row, uint32_t lane, LogitRow &r) {
    if (!p.start) {
        r = LogitRow{row, (int)row, 1};
        return row < p.sequences;
    }
    ErKv8Batch b = {};
    b.start = p.start;
    b.sequences = p.sequences;
    r.s = uniform(sequence_of_row(b, row, lane));
    if (r.s >= p.sequences) return false;
    const int rows = (int)p.rows;
    r.row0 = min(max(load_shared(p.start + r.s), 0), rows);
    r.n = min(max(min(load_shared(p.start + r.s + 1), rows) - r.row0, 0), (int)p.maxRows);
    return (int)row >= r.row0 && (int)row < r.row0 + r.n;
}

// One slice of one row.  How often the context has each token of the slice is
// counted in LDS, whole numbers whose order does not matter, and so is which
// entry of the biases is a token's last; then the logits pass once.  A value
// that a rule changes is formed in 64 bits and rounded once.
ER_DEV void choose_slice(const ErChooseArgs &p, uint32_t *lds) {
    const uint32_t row = blockIdx.x / p.slices, at = blockIdx.x % p.slices, tid = threadIdx.x, lane = tid & 63u;
    LogitRow r;
    if (!logit_row(p, row, lane, r)) return;
    const uint32_t from = at * p.slice, n = min(p.vocab - from, p.slice);
    double repetition = 1.0, presence = 0.0, frequency = 0.0;
    bool counts = false, biased = false;
    if (p.penalty) {
        const float *w = p.penalty + 3 * (size_t)r.s;
        const float a = load_shared(w), b = load_shared(w + 1), c = load_shared(w + 2);
        repetition = a, presence = b, frequency = c;
        counts = !(a == 1.0f && b == 0.0f && c == 0.0f);
    }
    const uint32_t known = counts && p.history ? min((uint32_t)max(load_shared(p.historyLen + r.s), 0), p.historyStride) : 0;
    const uint32_t drafts = counts && p.seen ? (uint32_t)r.n : 0;
    counts = known + drafts > 0;
    const uint32_t entries = p.bias ? min((uint32_t)max(load_shared(p.biasLen + r.s), 0), p.biasStride) : 0;
    biased = entries > 0;
    uint32_t *times = lds, *entry = lds + (p.penalty ? p.slice : 0);
    if (counts || biased) {
        for (uint32_t i = tid; i < p.slice; i += ER_CHOOSE_THREADS) {
            if (counts) times[i] = 0;
            if (biased) entry[i] = 0;
        }
        __syncthreads();
        for (uint32_t i = tid; i < known; i += ER_CHOOSE_THREADS) {
            const uint32_t t = (uint32_t)p.history[(size_t)r.s * p.historyStride + i] - from;
            if (t < n) atomicAdd(times + t, 1u);
        }
        for (uint32_t i = tid; i < drafts; i += ER_CHOOSE_THREADS) {
            const uint32_t word = p.seen[(size_t)row * p.words + (i >> 5)], t = (uint32_t)p.token[r.row0 + i] - from;
            if ((word >> (i & 31u) & 1u) && t < n) atomicAdd(times + t, 1u);
        }
        for (uint32_t i = tid; i < entries; i += ER_CHOOSE_THREADS) {
            const uint32_t t = (uint32_t)p.biasToken[(size_t)r.s * p.biasStride + i] - from;
            if (t < n) atomicMax(entry + t, i + 1);
        }
        __syncthreads();
    }
    const float *x = p.logits + (size_t)row * p.stride + from;
    float *y = p.out ? p.out + (size_t)row * p.stride + from : nullptr;
    const uint32_t *allowed = p.allowed ? p.allowed + (size_t)row * p.allowedStride + (from >> 5) : nullptr;
    const float *bias = p.bias + (size_t)r.s * p.biasStride;
    Candidate best = {-__builtin_inff(), ER_NO_TOKEN};
    for (uint32_t i = 4 * tid; i < n; i += 4 * ER_CHOOSE_THREADS) {
        const bool whole = i + 4 <= n;
        float v[4];
        if (whole) {
            const f32x4 w = *(const f32x4_a4 *)(x + i);
            v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) v[k] = i + k < n ? x[i + k] : 0.0f;
        }
        const uint32_t bits = allowed ? allowed[i >> 5] >> (i & 31u) : 15u;
        if (counts || biased) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t c = counts ? times[i + k] : 0u, e = biased ? entry[i + k] : 0u;
                if (c | e) {
                    double d = (double)v[k];
                    if (c) d = (d > 0.0 ? d / repetition : d * repetition) - (presence + frequency * (double)c);
                    if (e) d += (double)bias[e - 1];
                    v[k] = (float)d;
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const bool able = bits >> k & 1u;
            v[k] = able ? v[k] : -__builtin_inff();
            if (able && i + k < n) best = better(best, Candidate{v[k], from + i + k});
        }
        if (y) {
            if (whole) {
                *(f32x4_a4 *)(y + i) = f32x4{v[0], v[1], v[2], v[3]};
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)
                    if (i + k < n) y[i + k] = v[k];
            }
        }
    }
    if (!p.chosen) return;
    __shared__ Candidate waves[ER_CHOOSE_THREADS / 64];
    best = wave_best(best);
    if (lane == 63) waves[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int i = 1; i < ER_CHOOSE_THREADS / 64; ++i) waves[0] = better(waves[0], waves[i]);
        if (p.slices == 1) {
            p.chosen[row] = (int)waves[0].token;
        } else {
            p.partV[blockIdx.x] = waves[0].v;
            p.partI[blockIdx.x] = waves[0].token;
        }
    }
}

extern __shared__ __attribute__((aligned(16))) uint32_t er_choose_lds[];
extern "C" __global__ void __launch_bounds__(ER_CHOOSE_THREADS) er_choose_slices(ErChooseArgs p) { choose_slice(p, er_choose_lds); }

// The best of a row's slices: a wave a row.
extern "C" __global__ void __launch_bounds__(ER_CHOOSE_THREADS) er_choose_join(ErChooseArgs p) {
    const uint32_t row = uniform((blockIdx.x * ER_CHOOSE_THREADS + threadIdx.x) >> 6), lane = threadIdx.x & 63u;
    LogitRow r;
    if (row >= p.rows || !logit_row(p, row, lane, r)) return;
    Candidate best = {-__builtin_inff(), ER_NO_TOKEN};
    for (uint32_t i = lane; i < p.slices; i += 64)
        best = better(best, Candidate{p.partV[(size_t)row * p.slices + i], p.partI[(size_t)row * p.slices + i]});
    best = wave_best(best);
    if (lane == 63) p.chosen[row] = (int)best.token;
}
