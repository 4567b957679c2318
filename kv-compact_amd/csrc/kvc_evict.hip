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
    unsigned * keys;       // [groups][n][max_len]
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

__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 0;
    const unsigned u = __float_as_uint(x + 0.0f);   // (-0 is 0)
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Four cells a thread.
__global__ __launch_bounds__(256) void k_cell_keys(PickArgs p) {
    const int part = blockIdx.x % p.parts, i = blockIdx.x / p.parts % p.n, group = blockIdx.x / p.parts / p.n;
    const int cells = cells_of(p, i);
    if (cells <= 0) return;
    const int seq = p.seqs[i], start = p.start[i], len = start + cells;
    const int kept = p.keep[i] < cells ? p.keep[i] : cells;
    const int stay = len - (p.recent < kept ? p.recent : kept);
    const int l0 = p.groups == 1 ? 0 : group, l1 = p.groups == 1 ? p.n_layers : group + 1;
    for (int c = (part * 256 + (int)threadIdx.x) * 4; c < len; c += p.parts * 1024) {
        if (c + 4 <= start) continue;
        double sum[4] = {0, 0, 0, 0};
        float top[4] = {NAN, NAN, NAN, NAN};
        for (int l = l0; l < l1; l++) {
            const float * w = p.weight + ((long long)l * p.max_seqs + seq) * p.H * p.room + c;
            for (int h = 0; h < p.H; h++) {
                const float4 x = *reinterpret_cast<const float4 *>(w + h * p.room);   // (a row is whole pages)
                if (p.most) {
                    top[0] = fmaxf(top[0], x.x);
                    top[1] = fmaxf(top[1], x.y);
                    top[2] = fmaxf(top[2], x.z);
                    top[3] = fmaxf(top[3], x.w);
                } else {
                    sum[0] += x.x;
                    sum[1] += x.y;
                    sum[2] += x.z;
                    sum[3] += x.w;
                }
            }
        }
        unsigned * out = p.keys + ((long long)group * p.n + i) * p.max_len;
        for (int j = 0; j < 4; j++)
            if (c + j < len) out[c + j] = c + j >= stay ? kAlways : key_of(p.most ? top[j] : (float)sum[j]);
    }
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

// A block per request and group of layers.
__global__ __launch_bounds__(kPick) void k_pick(PickArgs p) {
    __shared__ int lds[kWaves], kept_of[kPick], first[kPick], bins[256];
    __shared__ long long sums[kWaves];
    __shared__ int found[2];
    const int t = threadIdx.x, i = blockIdx.x % p.n, group = blockIdx.x / p.n;
    // every block goes through the requests: what they keep (-1: refused), and where their indices begin
    int kept = -1;
    if (t < p.n) {
        const int cells = cells_of(p, t);
        kept = cells < 0 ? -1 : p.keep[t] < cells ? p.keep[t] : cells;
        if (kept > p.n_idx) kept = -1;
        for (int j = 0; j < t && kept >= 0; j++)
            if (p.seqs[j] == p.seqs[t]) kept = -1;
    }
    long long total;
    first[t] = (int)pick_scan((long long)(kept > 0 ? kept : 0), sums, &total);
    kept_of[t] = kept;
    __syncthreads();
    if (total > p.n_idx) {   // (rare) in order, each that still fits
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
    const int k = kept_of[i], to = first[i];
    if (group == 0 && t == 0) {
        p.status[i] = k < 0 ? KVC_REQ_BAD : 0;
        p.granted[i] = k < 0 ? -1 : p.seqs[i];
        p.cu[i + 1] = to + (k < 0 ? 0 : k);
        if (i == 0) p.cu[0] = 0;
    }
    if (k <= 0) return;
    const int start = p.start[i], len = p.len[p.seqs[i]];
    const unsigned * keys = p.keys + ((long long)group * p.n + i) * p.max_len;
    // the k-th largest key, a byte at a time
    unsigned top = 0;
    int left = k;   // of the keys that begin with top's bytes, how many are kept
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) bins[t] = 0;
        __syncthreads();
        for (int c = start + t; c < len; c += kPick) {
            const unsigned u = keys[c];
            if (shift == 24 || u >> (shift + 8) == top >> (shift + 8)) atomicAdd(&bins[u >> shift & 255], 1);
        }
        __syncthreads();
        if (t == 0) {
            int b = 255, more = left;
            while (more > bins[b]) more -= bins[b--];
            found[0] = b;
            found[1] = more;
        }
        __syncthreads();
        top |= (unsigned)found[0] << shift;
        left = found[1];
        __syncthreads();
    }
    int * out = p.idx + group * p.ld_idx + to;
    int done = 0, equal = 0;
    for (int c0 = start; c0 < len; c0 += kPick) {
        const int c = c0 + t;
        const unsigned u = c < len ? keys[c] : 0;
        const int same = c < len && u == top;
        int all;
        const int nth = equal + pick_scan(same, lds, &all);
        equal += all;
        const int stays = c < len && (u > top || (same && nth < left));
        const int where = done + pick_scan(stays, lds, &all);
        done += all;
        if (stays) out[where] = c - start;
    }
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
// the block reads is at or behind what it writes.
__global__ __launch_bounds__(256) void k_take_weights(TakeArgs p) {
    constexpr int STEP = 1024;
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
            bool ok[STEP / 256];
#pragma unroll
            for (int j = 0; j < STEP / 256; j++) {
                const int c = c0 + 256 * j + (int)threadIdx.x;
                const int a = c < kept ? idx[c] : -1;
                ok[j] = a >= c && (long long)lead + a < p.room;
                x[j] = ok[j] ? from[lead + a] : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < STEP / 256; j++)
                if (ok[j]) to[lead + c0 + 256 * j + (int)threadIdx.x] = x[j];
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
    return sizeof(unsigned) * (size_t)(a->ld_idx ? c->n_layers : 1) * n * pick_cells(c, a);
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
    p.n = n; p.n_idx = a->n_idx; p.recent = a->recent; p.max_len = pick_cells(c, a); p.max_seqs = c->max_seqs;
    p.H = c->n_head_kv; p.n_layers = c->n_layers; p.groups = a->ld_idx ? c->n_layers : 1; p.most = a->heads == KVC_HEADS_MAX;
    p.room = (long long)c->max_pages * c->page_size;
    const int units = p.groups * n;
    const int want = p.max_len / 1024 + 1, most = (1 << 22) / units;
    p.parts = want < most ? want : most;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    if (!launch(k_cell_keys, dim3((unsigned)(units * p.parts)), dim3(256), st, p) ||
        !launch(k_pick, dim3((unsigned)units), dim3(kPick), st, p))
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
