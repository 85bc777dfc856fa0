// The acceptance kernel (er_accept.hip) on the CPU, a workgroup's waves in an
// order of the caller's: whenever several can go on, the one that stands first in
// the order does, as far as its next barrier.  What a kernel leaves between two
// barriers to whichever wave is faster comes out otherwise in another order.
#include "er_draft.h"

#include <ucontext.h>

#include <cmath>
#include <cstdlib>
#include <cstring>
#include <vector>

#include <algorithm>
using std::max;
using std::min;

namespace {

constexpr int kWaves = ER_KV8_THREADS / 64;

enum class State { Ready, Lane, Barrier, Done };
struct Fiber {
    ucontext_t context;
    std::vector<char> stack;
    State state;
    uint32_t given;
};
Fiber g_fibers[ER_KV8_THREADS];
uint32_t g_given[kWaves][64];  // of a wave's last exchange
ucontext_t g_scheduler;
int g_now;
bool g_failed;
void (*g_kernel)();

struct Dim {
    uint32_t x;
};
Dim blockIdx, threadIdx;

void wait(State s) {
    const int me = g_now;
    g_fibers[me].state = s;
    swapcontext(&g_fibers[me].context, &g_scheduler);
    threadIdx.x = (uint32_t)me;
}
// Every lane gives a value and gets all of the wave's.
const uint32_t *exchange(uint32_t v) {
    g_fibers[g_now].given = v;
    wait(State::Lane);
    return g_given[threadIdx.x >> 6];
}
void start() {
    threadIdx.x = (uint32_t)g_now;
    g_kernel();
    g_fibers[g_now].state = State::Done;
    swapcontext(&g_fibers[g_now].context, &g_scheduler);
}

// One workgroup; false: its waves wait for each other for good.
bool run_workgroup(const int *order) {
    for (int i = 0; i < (int)ER_KV8_THREADS; ++i) {
        Fiber &f = g_fibers[i];
        f.stack.resize(64 << 10);
        f.state = State::Ready;
        getcontext(&f.context);
        f.context.uc_stack.ss_sp = f.stack.data();
        f.context.uc_stack.ss_size = f.stack.size();
        f.context.uc_link = &g_scheduler;
        makecontext(&f.context, start, 0);
    }
    auto all = [](int from, int n, State s) {
        for (int i = from; i < from + n; ++i)
            if (g_fibers[i].state != s) return false;
        return true;
    };
    while (true) {
        bool moved = false;
        for (int k = 0; k < kWaves && !moved; ++k) {
            const int first = 64 * order[k];
            if (all(first, 64, State::Lane)) {
                for (int i = 0; i < 64; ++i) {
                    g_given[order[k]][i] = g_fibers[first + i].given;
                    g_fibers[first + i].state = State::Ready;
                }
            }
            for (int i = 0; i < 64; ++i)
                if (g_fibers[first + i].state == State::Ready) {
                    moved = true;
                    g_now = first + i;
                    swapcontext(&g_scheduler, &g_fibers[g_now].context);
                }
        }
        if (moved) continue;
        if (all(0, ER_KV8_THREADS, State::Done)) return true;
        if (!all(0, ER_KV8_THREADS, State::Barrier)) return false;
        for (Fiber &f : g_fibers) f.state = State::Ready;
    }
}

// ---- what the kernel takes from the device's headers

#define ER_DEV inline
#define __global__
#define __shared__ static
#define __launch_bounds__(...)
#define __syncthreads() wait(State::Barrier)

uint64_t ballot(bool b) {
    const uint32_t *v = exchange(b);
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) r |= (uint64_t)(v[i] != 0) << i;
    return r;
}
#define __ballot ballot
int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }
int readlane(int v, int lane) { return (int)exchange((uint32_t)v)[lane]; }
#define __builtin_amdgcn_readlane readlane

// Of a value that has to be the same in all lanes.
int uniform(int v) {
    const uint32_t *all = exchange((uint32_t)v);
    for (int i = 0; i < 64; ++i) g_failed |= all[i] != all[0];
    return (int)all[0];
}
float as_float(uint32_t u) {
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}
uint32_t as_bits(float f) {
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return u;
}
#define __uint_as_float as_float
#define __float_as_uint as_bits
float wave_max(float v) {
    const uint32_t *all = exchange(as_bits(v));
    float m = as_float(all[0]);
    for (int i = 1; i < 64; ++i) m = std::fmax(m, as_float(all[i]));
    return m;
}

struct f32x2 {
    float x, y;
};
float value_of(uint32_t code) {
    const int e = (int)(code >> 3 & 15u), m = (int)(code & 7u);
    const float v = (code & 0x7fu) == 0x7fu ? NAN : e == 0 ? std::ldexp((float)m, -9) : std::ldexp((float)(8 + m), e - 10);
    return code & 0x80u ? -v : v;
}
uint32_t code_of(float v) {
    if (!std::isfinite(v)) return 0xffu;
    const double a = std::fabs((double)v);
    uint32_t best = 0;
    for (uint32_t c = 1; c < 0x7f; ++c) {
        const double near = std::fabs(value_of(c) - a), so_far = std::fabs(value_of(best) - a);
        if (near < so_far || (near == so_far && c % 2 == 0)) best = c;
    }
    return best | (std::signbit(v) ? 0x80u : 0u);
}
f32x2 cvt_pk_f32_fp8(int codes, bool high) {
    const uint32_t c = (uint32_t)codes >> (high ? 16 : 0);
    return {value_of(c & 0xffu), value_of(c >> 8 & 0xffu)};
}
#define __builtin_amdgcn_cvt_pk_f32_fp8 cvt_pk_f32_fp8
uint32_t codes4(float a, float b, float c, float d) { return code_of(a) | code_of(b) << 8 | code_of(c) << 16 | code_of(d) << 24; }
uint32_t recode4(uint32_t c, float f) {
    const f32x2 lo = cvt_pk_f32_fp8((int)c, false), hi = cvt_pk_f32_fp8((int)c, true);
    return codes4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
}
int block_exponent(float peak) {
    int e;
    const float m = std::frexp(peak, &e);
    return max(e - (m <= 0.875f ? 9 : 8), -100);
}
float exp2i(int j) { return std::ldexp(1.0f, j); }
float finite_magnitude(float v) { return std::isfinite(v) ? std::fabs(v) : 0.0f; }

struct Sequence {
    int row0, n, len;
};
Sequence sequence_of(const ErKv8Batch &b, uint32_t s) {
    Sequence q;
    q.row0 = min(max(b.start[s], 0), (int)b.rows);
    q.n = min(max(min(b.start[s + 1], (int)b.rows) - q.row0, 0), (int)b.maxRows);
    q.len = min(max(b.len[s], 0), (int)b.maxLen);
    return q;
}
int page_of(const ErKv8Batch &b, const ErKv8Cache &c, uint32_t s, int t) {
    const int p = b.table[(size_t)s * b.stride + ((uint32_t)t >> c.shift)];
    return (uint32_t)p < c.pages ? p : -1;
}

#include "er_accept.hip"

ErAcceptArgs g_args;
uint32_t g_width;
void kernel() {
    if (g_width == 64)
        er_kv8_accept_d64(g_args);
    else if (g_width == 128)
        er_kv8_accept_d128(g_args);
    else
        er_kv8_accept_d256(g_args);
}

}  // namespace

// pointers: codes and scales of keys, of values, table, lengths, starts, parent, token, chosen, path, count, next,
// left; sizes: pages, heads, log2 of a page's tokens, head width, sequences, table stride, rows, most rows, most
// tokens.  0: done; 1: values that all lanes should hold alike differ; 2: waves wait for good.
extern "C" int accept_in_order(void *const *at, const uint32_t *size, const int *order) {
    g_args = ErAcceptArgs{};
    g_args.c = ErKv8Cache{(uint8_t *)at[0], (uint8_t *)at[2], (float *)at[1], (float *)at[3], size[0], size[1], size[2]};
    g_args.b = ErKv8Batch{(const int32_t *)at[4], (const int32_t *)at[5], (const int32_t *)at[6], size[4], size[5], size[6], size[7], size[8]};
    g_args.parent = (const int32_t *)at[7], g_args.token = (const int32_t *)at[8], g_args.chosen = (const int32_t *)at[9];
    g_args.path = (int32_t *)at[10], g_args.count = (int32_t *)at[11], g_args.next = (int32_t *)at[12], g_args.left = (int32_t *)at[13];
    g_width = size[3];
    g_kernel = kernel;
    g_failed = false;
    for (blockIdx.x = 0; blockIdx.x < 2 * g_args.c.heads * g_args.b.sequences; ++blockIdx.x)
        if (!run_workgroup(order)) return 2;
    return g_failed ? 1 : 0;
}
