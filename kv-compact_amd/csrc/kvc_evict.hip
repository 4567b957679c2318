// Which cells of a sequence to keep by the weight they gathered, and weights
// that follow a fork or a compaction (include/kvc-cache.h: kvc_cache_pick,
// kvc_cache_take_weights).
//
// A cell's score is the sum of its heads' weights (in 64 bits, rounded once) or
// the largest of them, as an unsigned key that orders like it: 0 for NaN, all
// ones for the last cells, which stay whatever they gathered. The keep-th
// largest key is found by its bytes from the top, a histogram each; cells above
// it are kept, and of those equal to it the first.
#include "kvc_launch.h"

#include <stdint.h>

namespace kvc {

namespace {

constexpr int kPick = 1024;          // threads of a picking block
constexpr int kWaves = kPick / 64;
constexpr unsigned kAlways = ~0u;    // key of a cell that stays

struct PickArgs {
    const int * seqs;
    const int * start;
    const int * keep;
    const int * len;
    const float * weight;
    int * idx;
    long long ld_idx;
    int * cu;
    int * granted;
    int * status;
    unsigned * keys;       // [groups][n][stride]
    long long stride;      // max_len, in whole fours
    int n, n_idx, recent, max_len, max_seqs, H, n_layers, groups, most;
    int parts;             // blocks of a unit's keys
    long long room;        // cells of a row of weights
};

// Cells of a request, or a negative number: it is refused whatever the others are.
__device__ __forceinline__ int cells_of(const PickArgs & p, int i) {
    const int s = p.seqs[i];
    if (s < 0 || s >= p.max_seqs) return -1;
    const int len = p.len[s], start = p.start[i];
    return start < 0 || start > len || len > p.max_len || len > p.room || p.keep[i] < 0 ? -1 : len - start;
}

// (0 is left for what is no cell of the choice)
__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 1;
    const unsigned u = __float_as_uint(x + 0.0f);   // (-0 is 0)
    return u >> 31 ? ~u : u | 0x80000000u;
}

typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

// A request's cells as a unit works on them.
struct Unit {
    int seq, start, len, stay;   // cells at or past `stay` are kept whatever they gathered
    int l0, l1;                  // layers
    const float * weight;        // layer l0's, head 0
};
__device__ __forceinline__ Unit unit_of(const PickArgs & p, int seq, int start, int len, int group, int kept) {
    Unit u;
    u.seq = seq;
    u.start = start;
    u.len = len;
    u.stay = u.len - (p.recent < kept ? p.recent : kept);
    u.l0 = p.groups == 1 ? 0 : group;
    u.l1 = p.groups == 1 ? p.n_layers : group + 1;
    u.weight = p.weight + ((long long)u.l0 * p.max_seqs + u.seq) * p.H * p.room;
    return u;
}

// Keys of cells c .. c+3 (c a multiple of 4, below the length).
__device__ __forceinline__ u4 keys_at(const PickArgs & p, const Unit & u, int c) {
    u4 k = {0, 0, 0, 0};
    if (c + 4 <= u.start) return k;
    double sum[4] = {0, 0, 0, 0};
    f4 top = {NAN, NAN, NAN, NAN};
    for (int l = u.l0; l < u.l1; l++) {
        // (a row is whole pages: four cells at a time)
        const float * w = u.weight + (long long)(l - u.l0) * p.max_seqs * p.H * p.room + c;
        if (p.most) {
#pragma unroll 8
            for (int h = 0; h < p.H; h++) {
                const f4 x = *reinterpret_cast<const f4 *>(w + h * p.room);
#pragma unroll
                for (int j = 0; j < 4; j++) top[j] = fmaxf(top[j], x[j]);
            }
        } else {
#pragma unroll 8
            for (int h = 0; h < p.H; h++) {
                const f4 x = *reinterpret_cast<const f4 *>(w + h * p.room);
#pragma unroll
                for (int j = 0; j < 4; j++) sum[j] += x[j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (c + j >= u.start && c + j < u.len) k[j] = c + j >= u.stay ? kAlways : key_of(p.most ? top[j] : (float)sum[j]);
    return k;
}

// The keys by themselves, for few units of many cells. Four cells a thread.
__global__ __launch_bounds__(256) void k_cell_keys(PickArgs p) {
    const int part = blockIdx.x % p.parts, i = blockIdx.x / p.parts % p.n, group = blockIdx.x / p.parts / p.n;
    const int cells = cells_of(p, i);
    if (cells <= 0) return;
    const Unit u = unit_of(p, p.seqs[i], p.start[i], p.start[i] + cells, group, p.keep[i] < cells ? p.keep[i] : cells);
    u4 * out = reinterpret_cast<u4 *>(p.keys + ((long long)group * p.n + i) * p.stride);
    for (int c = (part * 256 + (int)threadIdx.x) * 4; c < u.len; c += p.parts * 1024) out[c >> 2] = keys_at(p, u, c);
}

// Sum of v over the block's threads before this one; *total the whole sum.
template <class T> __device__ T pick_scan(T v, T * lds, T * total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    T x = v;
    for (int o = 1; o < 64; o <<= 1) {
        const T y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) lds[w] = x;
    __syncthreads();
    T before = 0, all = 0;
    for (int j = 0; j < kWaves; j++) {
        before += j < w ? lds[j] : 0;
        all += lds[j];
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// Sum of v over the wave's lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// Request i: what it keeps (-1: it is refused) and where its indices begin, from
// all requests of the call, and its sequence's cells. Up to 64 by each wave by
// itself.
__device__ void plan_of(const PickArgs & p, int i, int & k, int & to, int & seq_i, int & start, int & len) {
    __shared__ long long sums[kWaves];
    __shared__ int ids[kPick], kept_of[kPick], first[kPick];
    const int t = p.n <= 64 ? threadIdx.x & 63 : threadIdx.x;
    int kept = -1, seq = -1, from = 0, cells = 0;
    if (t < p.n) {
        seq = p.seqs[t];
        from = p.start[t];
        cells = cells_of(p, t);
        kept = cells < 0 ? -1 : p.keep[t] < cells ? p.keep[t] : cells;
        if (kept > p.n_idx) kept = -1;
    }
    if (p.n <= 64) {
        seq_i = __shfl(seq, i);
        start = __shfl(from, i);
        len = start + __shfl(cells, i);
        for (int j = 0; j < p.n; j++) {
            const int other = __shfl(seq, j);   // (all lanes)
            if (j < t && other == seq) kept = -1;
        }
        long long at = kept > 0 ? kept : 0;
        const long long mine = at;
        for (int o = 1; o < 64; o <<= 1) {
            const long long y = __shfl_up(at, o);
            if (t >= o) at += y;
        }
        if (__shfl(at, 63) <= p.n_idx) {
            k = __shfl(kept, i);
            to = (int)__shfl(at - mine, i);
            return;
        }
        // (rare) in order, each that still fits
        int used = 0;
        for (int j = 0; j <= i; j++) {
            k = __shfl(kept, j);
            to = used;
            if (k > p.n_idx - used) k = -1;
            if (k > 0) used += k;
        }
        return;
    }
    ids[t] = seq;
    __syncthreads();
    for (int j = 0; j < t && kept >= 0; j++)
        if (ids[j] == seq) kept = -1;
    long long total;
    first[t] = (int)pick_scan((long long)(kept > 0 ? kept : 0), sums, &total);
    kept_of[t] = kept;
    __syncthreads();
    if (total > p.n_idx) {
        if (t == 0) {
            int used = 0;
            for (int j = 0; j < p.n; j++) {
                first[j] = used;
                if (kept_of[j] > p.n_idx - used) kept_of[j] = -1;
                if (kept_of[j] > 0) used += kept_of[j];
            }
        }
        __syncthreads();
    }
    k = kept_of[i];
    to = first[i];
    seq_i = ids[i];
    start = p.start[i];
    len = k < 0 ? 0 : p.len[seq_i];
}

// A block per request and group of layers. Its waves have neighbouring
// stretches of the cells, a thread four cells at a time, the same ones in every
// pass: what it writes it alone reads again. FUSED: the keys are worked out on
// the way of the first pass.
//
// The k-th largest key by its bits from the top. The first 11, sign, exponent
// and two bits more, spread the lanes of a wave over a histogram in LDS where
// eight bits would not. The keys that share those of the k-th one, mostly a few
// hundred, are then listed in LDS with their wave, and the other 21 bits and each
// wave's counts come from the list: three passes over the cells in all. Where
// they are too many for the list, the passes go on over all cells.
//
// 20 % of 16 sequences of up to 32768 cells, 32 layers, 8 heads: 98 us, 70 of them
// the read of the weights (313 MB, 4.5 TB/s; the longest sequences' blocks), then
// the search, in which all blocks are at once. One sequence of 5120 cells: 15 us,
// a chain of latencies (passes over L2, barriers).
constexpr int kList = 4096;

template <bool FUSED> __global__ __launch_bounds__(kPick, 8) void k_pick(PickArgs p) {
    __shared__ int lds[kWaves], bins[2048], found[3], above[kWaves], same[kWaves], listed;
    __shared__ unsigned list[kList];   // low 21 bits of a key, and the wave
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // (a request's blocks on different dies and CUs: requests differ in length)
    const int group = blockIdx.x / p.n, i = (blockIdx.x % p.n + group + group / 8) % p.n;
    int k, to, seq, start, len;
    plan_of(p, i, k, to, seq, start, len);
    if (group == 0 && t == 0) {
        p.status[i] = k < 0 ? KVC_REQ_BAD : 0;
        p.granted[i] = k < 0 ? -1 : seq;
        p.cu[i + 1] = to + (k < 0 ? 0 : k);
        if (i == 0) p.cu[0] = 0;
    }
    if (k <= 0) return;
    const Unit u = unit_of(p, seq, start, len, group, k);
    const int turns = (u.len + 4 * kPick - 1) / (4 * kPick);   // of 256 cells a wave
    const int c0 = wave * turns * 256 + 4 * lane;
    u4 * keys = reinterpret_cast<u4 *>(p.keys + ((long long)group * p.n + i) * p.stride);

    // one more in place b of the histogram, of the lanes that are `in` (all lanes call)
    auto count = [&](bool in, int b) {
        // (many alike: one addition for the lanes that agree with the first)
        const unsigned long long who = __ballot(in);
        if (!who) return;
        const int lead = __ffsll((long long)who) - 1, b0 = __builtin_amdgcn_readlane(b, lead);
        const unsigned long long with = __ballot(in && b == b0);
        if (lane == lead) atomicAdd(&bins[b0], __popcll(with));
        if (in && b != b0) atomicAdd(&bins[b], 1);
    };
    auto clear = [&] {
        bins[t] = 0;
        bins[t + kPick] = 0;
        __syncthreads();
    };
    unsigned top = 0;
    int left = k;   // of the keys that begin with top's bits, how many are kept
    // the place of the histogram that the left-th largest is in; how many are in it
    // (not read from bins: a wave ahead may be clearing them)
    auto find = [&](int shift) {
        __syncthreads();
        // from the top: thread t has places 2 t and 2 t + 1
        const int n0 = bins[2047 - 2 * t], n1 = bins[2046 - 2 * t];
        const int incl = wave_scan(n0 + n1);
        if (lane == 63) lds[wave] = incl;
        __syncthreads();
        int before = incl - n0 - n1;
#pragma unroll
        for (int j = 0; j < kWaves; j++) before += j < wave ? lds[j] : 0;
        if (before < left && left <= before + n0 + n1) {
            const bool second = left > before + n0;
            found[0] = 2047 - 2 * t - second;
            found[1] = left - before - (second ? n0 : 0);
            found[2] = second ? n1 : n0;
        }
        __syncthreads();
        top |= (unsigned)found[0] << shift;
        left = found[1];
        return found[2];
    };
    // f(four keys, their first cell) in ascending order (all lanes), the next four on their way
    auto each = [&](auto f) {
        u4 next = {0, 0, 0, 0};
        if (c0 < u.len) next = keys[c0 >> 2];
        for (int y = 0; y < turns; y++) {
            const u4 x = next;
            const int c = c0 + 256 * y;
            next = u4{0, 0, 0, 0};
            if (y + 1 < turns && c + 256 < u.len) next = keys[(c + 256) >> 2];
            f(x, c);
        }
    };
    const unsigned long long before_me = (1ull << lane) - 1;
    if (t == 0) listed = 0;
    if (t < kWaves) above[t] = same[t] = 0;
    clear();
    for (int y = 0; y < turns; y++) {
        const int c = c0 + 256 * y;
        u4 x = {0, 0, 0, 0};
        if (c < u.len) {
            if constexpr (FUSED) {
                x = keys_at(p, u, c);
                keys[c >> 2] = x;
            } else {
                x = keys[c >> 2];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) count(x[j] != 0, x[j] >> 21);
    }
    const int near = find(21);   // (uniform) keys that begin like the k-th
    int n_above = 0, n_same = 0;
    if (near <= kList) {
        each([&](u4 x, int) {
            bool in[4];
            unsigned long long who[4];
            int n = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                n_above += __popcll(__ballot(x[j] >> 21 > top >> 21));
                in[j] = x[j] != 0 && x[j] >> 21 == top >> 21;
                who[j] = __ballot(in[j]);
                n += __popcll(who[j]);
            }
            if (!n) return;
            int at = 0;
            if (lane == 0) at = atomicAdd(&listed, n);
            at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (in[j]) list[at + __popcll(who[j] & before_me)] = (x[j] & 0x1fffff) | (unsigned)wave << 21;
                at += __popcll(who[j]);
            }
        });
        for (int pass = 1; pass < 3; pass++) {
            const int shift = pass == 1 ? 10 : 0, bits = pass == 1 ? 11 : 10;
            clear();
            for (int e = t; e < kList; e += kPick) {
                const unsigned x = e < near ? list[e] & 0x1fffff : 0;
                count(e < near && x >> (shift + bits) == (top & 0x1fffff) >> (shift + bits), x >> shift & ((1 << bits) - 1));
            }
            find(shift);
        }
        for (int e = t; e < near; e += kPick) {
            const unsigned x = list[e] & 0x1fffff;
            if (x > (top & 0x1fffff)) atomicAdd(&above[list[e] >> 21], 1);
            if (x == (top & 0x1fffff)) atomicAdd(&same[list[e] >> 21], 1);
        }
        if (lane == 0) atomicAdd(&above[wave], n_above);
    } else {
        for (int pass = 1; pass < 3; pass++) {
            const int shift = pass == 1 ? 10 : 0, bits = pass == 1 ? 11 : 10;
            clear();
            each([&](u4 x, int) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    count(x[j] != 0 && x[j] >> (shift + bits) == top >> (shift + bits), x[j] >> shift & ((1 << bits) - 1));
            });
            find(shift);
        }
        each([&](u4 x, int) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                n_above += __popcll(__ballot(x[j] > top));
                n_same += __popcll(__ballot(x[j] == top));
            }
        });
        if (lane == 0) {
            above[wave] = n_above;
            same[wave] = n_same;
        }
    }
    __syncthreads();
    int done = 0, equal = 0;   // kept, and equal to top, before this wave's cells
    for (int j = 0; j < wave; j++) {
        done += above[j];
        equal += same[j];
    }
    done += equal < left ? equal : left;
    int * out = p.idx + group * p.ld_idx + to;
    each([&](u4 x, int c) {
        int nth = equal, where = done;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned long long alike = __ballot(x[j] == top);
            nth += __popcll(alike & before_me);
            equal += __popcll(alike);
        }
        bool stays[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            stays[j] = x[j] > top || (x[j] == top && nth < left);
            nth += x[j] == top;
            const unsigned long long kept = __ballot(stays[j]);
            where += __popcll(kept & before_me);
            done += __popcll(kept);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (stays[j]) out[where++] = c + j - u.start;
    });
}

struct TakeArgs {
    const int * src;
    const int * dst;
    const int * start;
    const int * cu;        // nullptr: all cells of dst
    const int * idx;
    long long ld_idx;
    const int * status;
    const int * len;
    float * weight;
    int n, n_idx, max_seqs, H, n_layers;
    long long room;
};

// A block per request, layer and head. Places are filled in ascending order and
// no cell moves down, so that a row can be moved within itself: what a step of
// the block reads is at or behind what it writes. A step is 16 cells a thread:
// two rounds of loads in all for most budgets. Bound by HBM: picking a fifth of
// the cells touches nearly every line, so that what 16 sequences of up to 32768
// cells keep, 32 layers of 8 heads, takes 85 us: 400 MB, 4.7 TB/s.
__global__ __launch_bounds__(256) void k_take_weights(TakeArgs p) {
    constexpr int STEP = 4096;
    for (long long u = blockIdx.x; u < (long long)p.n * p.n_layers * p.H; u += gridDim.x) {
        const int h = (int)(u % p.H), l = (int)(u / p.H % p.n_layers), i = (int)(u / p.H / p.n_layers);
        const int src = p.src[i], dst = p.dst[i];
        if (src < 0 || src >= p.max_seqs || dst < 0 || dst >= p.max_seqs || (p.status && p.status[i] != 0)) continue;
        int lead, kept = 0, k0 = 0;
        if (p.cu) {
            lead = p.start[i];
            k0 = p.cu[i];
            const long long k = (long long)p.cu[i + 1] - k0;
            if (lead < 0 || k0 < 0 || k < 0 || p.cu[i + 1] > p.n_idx || lead + k > p.room) continue;
            kept = (int)k;
        } else {
            lead = p.len[dst];
            if (lead < 0 || lead > p.room) continue;
        }
        const float * from = p.weight + (((long long)l * p.max_seqs + src) * p.H + h) * p.room;
        float * to = p.weight + (((long long)l * p.max_seqs + dst) * p.H + h) * p.room;
        if (src != dst)
            for (int c = threadIdx.x; c < lead; c += 256) to[c] = from[c];
        const int * idx = p.idx + l * p.ld_idx + k0;
        for (int c0 = 0; c0 < kept; c0 += STEP) {
            float x[STEP / 256];
            int at[STEP / 256];
#pragma unroll
            for (int j = 0; j < STEP / 256; j++) {
                const int c = c0 + 256 * j + (int)threadIdx.x;
                at[j] = c < kept ? idx[c] : -1;
            }
#pragma unroll
            for (int j = 0; j < STEP / 256; j++) {
                const int c = c0 + 256 * j + (int)threadIdx.x;
                if (at[j] < c || (long long)lead + at[j] >= p.room) at[j] = -1;
                x[j] = at[j] >= 0 ? from[lead + at[j]] : 0.0f;
            }
            if (src == dst) __syncthreads();
#pragma unroll
            for (int j = 0; j < STEP / 256; j++)
                if (at[j] >= 0) to[lead + c0 + 256 * j + (int)threadIdx.x] = x[j];
        }
        __syncthreads();
    }
}

int check_requests(int n) {
    if (n < 0) return -2;
    return n > KVC_CACHE_MAX_REQUESTS ? KV_COMPACT_E_UNSUPPORTED : 0;
}

int check_pick(const kvc_cache * c, int n, const kvc_pick_args * a) {
    if (int rc = check_cache(c)) return rc;
    if (!a) return -1;
    if (int rc = check_requests(n)) return rc;
    if (a->n_idx < 0 || a->recent < 0 || a->max_len < 0 || a->ld_idx < 0 ||
        (a->ld_idx && a->ld_idx < a->n_idx) ||
        (a->heads != KVC_HEADS_SUM && a->heads != KVC_HEADS_MAX))
        return -2;
    return (long long)(a->ld_idx ? c->n_layers : 1) * n >= 1 << 22 ? KV_COMPACT_E_UNSUPPORTED : 0;   // (a launch's threads)
}

// (no sequence holds more cells than its table row has)
int pick_cells(const kvc_cache * c, const kvc_pick_args * a) {
    const long long room = (long long)c->max_pages * c->page_size;
    return a->max_len < room ? a->max_len : (int)room;
}

}  // namespace

}  // namespace kvc

using namespace kvc;

extern "C" {

size_t kvc_cache_pick_workspace(const kvc_cache * c, int n, const kvc_pick_args * a) {
    if (check_pick(c, n, a) || n == 0) return 0;
    return sizeof(unsigned) * (size_t)(a->ld_idx ? c->n_layers : 1) * n * ((pick_cells(c, a) + 3LL) & ~3LL);
}

int kvc_cache_pick(const kvc_cache * c, int n, const kvc_pick_args * a, void * ws, size_t ws_bytes, void * stream) {
    if (int rc = check_pick(c, n, a)) return rc;
    if (n == 0) return 0;
    if (!a->seqs || !a->start || !a->keep || !a->weight || !a->cu || !a->granted || !a->status || (a->n_idx && !a->idx)) return -1;
    if (reinterpret_cast<uintptr_t>(a->weight) & 15) return KV_COMPACT_E_UNSUPPORTED;
    const size_t need = kvc_cache_pick_workspace(c, n, a);
    if (need && !ws) return -1;
    if (need && reinterpret_cast<uintptr_t>(ws) & 15) return KV_COMPACT_E_UNSUPPORTED;
    if (need > ws_bytes) return KVC_E_SCRATCH;
    PickArgs p{};
    p.seqs = a->seqs; p.start = a->start; p.keep = a->keep; p.len = c->len; p.weight = a->weight;
    p.idx = a->idx; p.ld_idx = a->ld_idx; p.cu = a->cu; p.granted = a->granted; p.status = a->status;
    p.keys = static_cast<unsigned *>(ws);
    p.stride = (pick_cells(c, a) + 3LL) & ~3LL;
    p.n = n; p.n_idx = a->n_idx; p.recent = a->recent; p.max_len = pick_cells(c, a); p.max_seqs = c->max_seqs;
    p.H = c->n_head_kv; p.n_layers = c->n_layers; p.groups = a->ld_idx ? c->n_layers : 1; p.most = a->heads == KVC_HEADS_MAX;
    p.room = (long long)c->max_pages * c->page_size;
    const int units = p.groups * n;
    const long long want = p.max_len / 1024 + 1, most = (1 << 22) / units;
    p.parts = (int)(want < most ? want : most);
    // Keys by the picking blocks themselves, or by a launch of their own where
    // those blocks are few and long: 32 layers, 20 % of one sequence kept and its
    // weights moved, us (own launch, picking blocks): 5120 cells 20.6 and 20.0,
    // 16384 30.6 and 36.7, 32768 48.6 and 63.9; 4 of up to 32768 79 both, 8 103
    // both, 16 of up to 8192 62.3 and 54.1. One list for all layers has a block a
    // request, and a thread adds layers x heads: 32 layers of 8, 5120 cells 31.4 and
    // 175, 16 of up to 8192 57.4 and 204, 256 of up to 2048 306 and 373; 8 layers 5120
    // cells 21.9 and 34.2; 2 layers 2000 cells 17.8 and 17.1.
    const bool alone = p.groups == 1 && p.n_layers > 1;
    const bool fused = !alone && (units >= 256 || p.max_len <= 8192);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    if (fused) return launch(k_pick<true>, dim3((unsigned)units), dim3(kPick), st, p) ? 0 : KV_COMPACT_E_DEVICE;
    if (!launch(k_cell_keys, dim3((unsigned)(units * p.parts)), dim3(256), st, p) ||
        !launch(k_pick<false>, dim3((unsigned)units), dim3(kPick), st, p))
        return KV_COMPACT_E_DEVICE;
    return 0;
}

int kvc_cache_take_weights(const kvc_cache * c, int n, const int * src, const int * dst, const int * start, const int * cu,
                           int n_idx, const int * idx, long long ld_idx, const int * status, float * weight, void * stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_requests(n)) return rc;
    if (n_idx < 0 || ld_idx < 0) return -2;
    if (n == 0) return 0;
    if (!src || !dst || !weight || (cu && (!start || (n_idx && !idx)))) return -1;
    if (reinterpret_cast<uintptr_t>(weight) & 3) return KV_COMPACT_E_UNSUPPORTED;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    TakeArgs p{src, dst, start, cu, idx, ld_idx, status, c->len, weight, n, n_idx, c->max_seqs, c->n_head_kv, c->n_layers,
               (long long)c->max_pages * c->page_size};
    const long long units = (long long)n * c->n_layers * c->n_head_kv;
    return launch(k_take_weights, dim3((unsigned)(units < 1 << 20 ? units : 1 << 20)), dim3(256), st, p) ? 0 : KV_COMPACT_E_DEVICE;
}

}  // extern "C"
