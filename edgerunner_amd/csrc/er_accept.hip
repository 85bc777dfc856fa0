// er_accept.hip -- acceptance of drafted tokens (part of er_draft.hip).

// The walk down a sequence's tree: from row 0 on to the lowest later row whose
// parent is the present one and whose token was chosen there, until there is
// none.  Up to 64 rows lie in a wave's lanes, and a step is a lane read and a
// ballot; more are taken 64 at a time from LDS.  path[] gets the rows.
struct Walk {
    int count, first, next;  // rows, the first that changes its place (count if none), the token chosen at the last
};
ER_DEV Walk walk(const ErAcceptArgs &p, const Sequence &q, const int *parent, const int *token, const int *chosen, int *path,
                 int lane) {
    Walk w = {0, 0, -1};
    int cur = 0;
    const bool few = q.n <= 64;
    int up = -1, tok = -1, pick = -1;
    if (few && lane < q.n) {
        up = parent[lane];
        tok = token[lane];
        pick = chosen[lane];
    }
    while (true) {
        if (lane == 0) path[w.count] = cur;
        w.first += cur == w.count && w.first == w.count ? 1 : 0;
        ++w.count;
        w.next = few ? __builtin_amdgcn_readlane(pick, cur) : uniform(chosen[cur]);
        int found = -1;
        if (few) {
            const uint64_t at = __ballot(up == cur && tok == w.next && lane > cur);
            if (at) found = __ffsll((unsigned long long)at) - 1;
        } else {
            for (int i = cur & ~63; i < q.n && found < 0; i += 64) {
                const int r = i + lane;
                const uint64_t at = __ballot(r < q.n && r > cur && parent[min(r, q.n - 1)] == cur && token[min(r, q.n - 1)] == w.next);
                if (at) found = i + __ffsll((unsigned long long)at) - 1;
            }
        }
        if (found < 0 || w.next < 0) return w;
        cur = found;  // larger than before, so the walk ends
    }
}

// The scale that codes of magnitude m (finite, in codes' own units) under the scale f ask for by the append's rule.
// The value m * f is not formed: 256 under 2^120, which an append leaves for values next to fp32's largest, is past
// them.  A value that is not finite asks for the least.
ER_DEV float scale_for(float m, float f) {
    const uint32_t u = __float_as_uint(f);
    if (m == 0.0f || finite_magnitude(f) == 0.0f) return exp2i(-100);
    const int j = block_exponent(m * __uint_as_float((u & 0x7fffffu) | 0x3f800000u)) + (int)(u >> 23) - 127;
    return exp2i(min(max(j, -100), 127));
}

// One workgroup takes the keys or values of one sequence and head; each walks
// for itself, the first of a sequence also writes the path.  Kept tokens that
// change their place are appended anew, page by page in ascending order, as
// the values that their codes stand for: all of a page's are read before any
// is written, and a kept token moves down, so that no page is written before
// the last read from it.  Bound by the chain of loads: starts, tree, table,
// codes; 4.6 us for one user's 26 drafts, 4.9 for 64 users', of which a call is
// most.
template <int D, int P>
ER_DEV void accept_moves(const ErAcceptArgs &p, const Sequence &q, uint32_t s, uint32_t head, bool values, const Walk &w,
                         const int *path, float (*needs)[4]) {
    constexpr int LANES = D / 4;                                                     // lanes a token
    constexpr int TOKENS = ER_KV8_THREADS / LANES < P ? ER_KV8_THREADS / LANES : P;  // tokens a pass
    constexpr int PASSES = P / TOKENS;
    const uint32_t H = p.c.heads, tid = threadIdx.x;
    const int base = q.len - q.n, first = max(base + w.first, 0), last = base + w.count;
    uint8_t *codes = values ? p.c.v : p.c.k;
    float *scales = values ? p.c.vs : p.c.ks;
    const int lane = (int)(tid % LANES), at = (int)(tid / LANES);
    uint32_t turn = 0;
    for (int begin = first & ~(P - 1); begin < last; begin += P) {
        const int t0 = max(first, begin), t1 = min(last, begin + P);
        const int page = uniform(page_of(p.b, p.c, s, begin));
        if (page < 0) continue;
        // Only a page that goes on to the barrier takes the other copy of the needs: two uses of a copy have a barrier between.
        turn ^= 1u;
        uint32_t c[PASSES];
        float f[PASSES];  // -1: nothing to write
        float need = 0.0f;  // the largest scale that a token asks for; 0: none has come
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int t = begin + i * TOKENS + at;
            f[i] = -1.0f;
            c[i] = 0;
            if (at < TOKENS && t >= t0 && t < t1) {
                const int from = base + path[t - base], source = page_of(p.b, p.c, s, from);
                if (source >= 0) {
                    const size_t block = (size_t)source * H + head;
                    c[i] = *(const uint32_t *)(codes + (block * P + (uint32_t)from % P) * D + 4 * lane);
                    f[i] = scales[block];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            if (f[i] < 0.0f) continue;
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
            const float m = fmaxf(fmaxf(finite_magnitude(lo.x), finite_magnitude(lo.y)),
                                  fmaxf(finite_magnitude(hi.x), finite_magnitude(hi.y)));
            need = fmaxf(need, scale_for(m, f[i]));
        }
        need = wave_max(need);
        if ((tid & 63u) == 0) needs[turn][tid >> 6] = need;
        const size_t block = (size_t)page * H + head;
        uint8_t *to = codes + block * (size_t)(P * D);
        const float old = t0 > begin ? scales[block] : 0.0f;
        __syncthreads();
        need = fmaxf(fmaxf(needs[turn][0], needs[turn][1]), fmaxf(needs[turn][2], needs[turn][3]));
        if (need == 0.0f) continue;  // none of the page's tokens has a page of its own
        const float now = fmaxf(old, need);
        if (now > old && t0 > begin) {
            const float g = old / now;
            for (uint32_t i = tid; i < (uint32_t)(t0 - begin) * (D / 4); i += ER_KV8_THREADS) {
                uint32_t *x = (uint32_t *)to + i;
                *x = recode4(*x, g);
            }
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            if (f[i] < 0.0f) continue;
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
            const float g = f[i] / now;  // scales are powers of two
            *((uint32_t *)(to + (i * TOKENS + at) * D) + lane) = codes4(lo.x * g, lo.y * g, hi.x * g, hi.y * g);
        }
        if (tid == 0) scales[block] = now;
    }
}

template <int D>
ER_DEV void kv8_accept(const ErAcceptArgs &p) {
    __shared__ int parent[ER_MOST_DRAFTS], token[ER_MOST_DRAFTS], chosen[ER_MOST_DRAFTS], path[ER_MOST_DRAFTS];
    __shared__ float needs[2][4];
    __shared__ Walk walked;
    const uint32_t H = p.c.heads, tid = threadIdx.x;
    const uint32_t part = blockIdx.x % (2 * H), s = blockIdx.x / (2 * H), head = part >> 1;
    const bool values = part & 1u, writes = part == 0;
    const Sequence q = sequence_of(p.b, s);
    if (q.n == 0) {
        if (writes && tid == 0) {
            p.count[s] = 0;
            p.next[s] = -1;
            p.left[s] = q.len;
        }
        return;
    }
    for (int i = (int)tid; i < q.n; i += ER_KV8_THREADS) {
        parent[i] = p.parent[q.row0 + i];
        token[i] = p.token[q.row0 + i];
        chosen[i] = p.chosen[q.row0 + i];
    }
    __syncthreads();
    if (tid < 64) {
        const Walk w = walk(p, q, parent, token, chosen, path, (int)tid);
        if (tid == 0) walked = w;
    }
    __syncthreads();
    const Walk w = {uniform(walked.count), uniform(walked.first), uniform(walked.next)};
    if (writes) {
        for (int i = (int)tid; i < q.n; i += ER_KV8_THREADS) p.path[q.row0 + i] = i < w.count ? path[i] : -1;
        if (tid == 0) {
            p.count[s] = w.count;
            p.next[s] = w.next;
            p.left[s] = max(q.len - q.n + w.count, 0);
        }
    }
    if (w.first == w.count) return;
    if (p.c.shift == 4)
        accept_moves<D, 16>(p, q, s, head, values, w, path, needs);
    else if (p.c.shift == 5)
        accept_moves<D, 32>(p, q, s, head, values, w, path, needs);
    else
        accept_moves<D, 64>(p, q, s, head, values, w, path, needs);
}

#define ER_KV8_ACCEPT(D)                                                                                           \
    extern "C" __global__ void __launch_bounds__(ER_KV8_THREADS) er_kv8_accept_d##D(ErAcceptArgs p) {              \
        kv8_accept<D>(p);                                                                                          \
    }
ER_KV8_ACCEPT(64)
ER_KV8_ACCEPT(128)
ER_KV8_ACCEPT(256)
