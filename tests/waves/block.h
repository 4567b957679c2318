// A kernel's own source on the CPU, lane by lane: every lane of a block is a
// coroutine, a wave's lanes meet at each cross-lane operation, and the waves
// meet at __syncthreads only. Between two block barriers one wave runs as far
// as it goes before the next starts, in the order that run_block is told, so
// that a value which passes between waves without a barrier is read stale or
// overwritten every time. LDS arrays are statics, which the undefined-behaviour
// sanitizer bounds.
#pragma once

#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

namespace {

struct Dim { unsigned x, y, z; };
enum Meet { NONE, WAVE, BLOCK };
struct Post { unsigned a, b; };
struct Lane {
    Dim tid;
    ucontext_t ctx;
    std::vector<char> stack;
    Meet at = NONE;
    bool done = false;
    unsigned ops = 0;   // cross-lane operations so far
};
std::vector<Lane> lanes;
Lane * cur;
ucontext_t sched;
Dim blockIdx, gridDim;
Post posted[16][2][64];   // [wave][parity of the operation][lane]
std::function<void()> kernel_body;

void meet(Meet m) {
    cur->at = m;
    swapcontext(&cur->ctx, &sched);
}
// every lane's values of this operation (a lane is at most one operation ahead)
const Post * gather(unsigned a, unsigned b = 0) {
    Post * p = posted[cur->tid.x >> 6][cur->ops++ & 1];
    p[cur->tid.x & 63] = {a, b};
    meet(WAVE);
    return p;
}
int lane_of() { return cur->tid.x & 63; }

unsigned __float_as_uint(float f) { unsigned i; memcpy(&i, &f, 4); return i; }
float __uint_as_float(unsigned i) { float f; memcpy(&f, &i, 4); return f; }
int __popcll(unsigned long long v) { return __builtin_popcountll(v); }
int __ffsll(long long v) { return __builtin_ffsll(v); }
unsigned __umul24(unsigned a, unsigned b) { return (a & 0xffffff) * (b & 0xffffff); }
unsigned long long __ballot(bool b) {
    const Post * p = gather(b);
    unsigned long long m = 0;
    for (int l = 0; l < 64; l++) m |= (unsigned long long)p[l].a << l;
    return m;
}
template <class T> T from_lane(T v, int l) {
    static_assert(sizeof(T) == 4 || sizeof(T) == 8, "");
    unsigned w[2] = {0, 0};
    memcpy(w, &v, sizeof(T));
    const Post p = gather(w[0], w[1])[l];
    w[0] = p.a;
    w[1] = p.b;
    memcpy(&v, w, sizeof(T));
    return v;
}
template <class T> T __shfl(T v, int l) { return from_lane(v, l & 63); }
template <class T> T __shfl_xor(T v, int o) { return from_lane(v, lane_of() ^ o); }
template <class T> T __shfl_up(T v, int o) { return from_lane(v, lane_of() >= o ? lane_of() - o : lane_of()); }
template <class T> T atomicAdd(T * p, T v) { const T was = *p; *p += v; return was; }
void __syncthreads() { meet(BLOCK); }

// What lane l takes in a data-parallel move (16 lanes a row), -1: nothing.
int dpp_from(int l, int ctrl) {
    const int row = l & ~15, m = l & 15;
    if (ctrl < 0x100) return (l & ~3) | (ctrl >> 2 * (l & 3) & 3);                       // a choice within four
    if (ctrl >= 0x111 && ctrl <= 0x11f) return m >= (ctrl & 15) ? l - (ctrl & 15) : -1;  // row shift right
    if (ctrl >= 0x121 && ctrl <= 0x12f) return row | ((m - (ctrl & 15)) & 15);           // row rotation
    if (ctrl == 0x141) return (l & ~7) | (7 - (l & 7));                                  // halves of a row mirrored
    if (ctrl == 0x142) return row >= 16 ? row - 1 : -1;                                  // a row's last lane to the next
    if (ctrl == 0x143) return l >= 32 ? 31 : -1;                                         // lane 31 to the upper half
    fprintf(stderr, "data-parallel move %x is not modelled\n", ctrl);
    exit(5);
}
int dpp_move(int old, int v, int ctrl, int rows, bool zero) {
    const Post * p = gather((unsigned)v);
    if (!(rows >> (lane_of() >> 4) & 1)) return old;
    const int from = dpp_from(lane_of(), ctrl);
    return from >= 0 ? (int)p[from].a : zero ? 0 : old;
}

#define __device__
#define __global__
#define __forceinline__ inline
#define __shared__ static
#define __align__(n) __attribute__((aligned(n)))
#define __launch_bounds__(...)
#define threadIdx (cur->tid)
#define __builtin_amdgcn_readlane(v, l) from_lane((int)(v), l)
#define __builtin_amdgcn_readfirstlane(v) from_lane((int)(v), 0)
#define __builtin_amdgcn_update_dpp(old, v, ctrl, rows, banks, zero) dpp_move(old, v, ctrl, rows, zero)

void lane_body() {
    kernel_body();
    cur->done = true;
    swapcontext(&cur->ctx, &sched);
}

// wave w to its next block barrier or its end; false: its lanes are at different operations
bool run_wave(int w) {
    for (;;) {
        int at[3] = {0, 0, 0}, done = 0;
        for (int l = 0; l < 64; l++) {
            Lane & x = lanes[64 * w + l];
            cur = &x;
            x.at = NONE;
            swapcontext(&sched, &x.ctx);
            done += x.done;
            at[x.at]++;
        }
        if (done == 64 || at[BLOCK] == 64) return true;
        if (at[WAVE] != 64) return false;
    }
}

// One block of `waves` waves, wave `first` the first to run behind each barrier (-1: from the last one down).
void run_block(int waves, int first, std::function<void()> f) {
    kernel_body = f;
    lanes.resize(64 * waves);
    for (unsigned t = 0; t < lanes.size(); t++) {
        Lane & x = lanes[t];
        x.tid = {t, 0, 0};
        x.done = false;
        x.ops = 0;
        x.stack.resize(128 << 10);
        getcontext(&x.ctx);
        x.ctx.uc_stack.ss_sp = x.stack.data();
        x.ctx.uc_stack.ss_size = x.stack.size();
        makecontext(&x.ctx, lane_body, 0);
    }
    for (int ended = 0; ended < waves;) {
        ended = 0;
        for (int k = 0; k < waves; k++) {
            const int w = first < 0 ? waves - 1 - k : (first + k) % waves;
            if (!run_wave(w)) {
                fprintf(stderr, "wave %d: lanes at different operations\n", w);
                exit(3);
            }
            ended += lanes[64 * w].done;
        }
        if (ended && ended < waves) {
            fprintf(stderr, "%d of %d waves ended, the others wait at a barrier\n", ended, waves);
            exit(4);
        }
    }
}

template <class T> std::vector<T> take(size_t n) {   // from stdin
    std::vector<T> v(n);
    if (n && fread(v.data(), sizeof(T), n, stdin) != n) exit(2);
    return v;
}
template <class T> void give(const std::vector<T> & v) { fwrite(v.data(), sizeof(T), v.size(), stdout); }

}  // namespace
