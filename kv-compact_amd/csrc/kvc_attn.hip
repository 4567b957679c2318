// Attention's entry points (include/kvc-cache.h): what is refused, which kernel
// a call takes and in how many key ranges, and the join of the ranges. The
// kernels themselves are in kvc_attn_kernels.h; those with a window are compiled
// in kvc_window.hip.
#include "kvc_attn_kernels.h"

#include <math.h>

#pragma clang fp contract(fast)

namespace kvc {

namespace {

// Joins the key ranges: W waves a row, a lane a range for the weights (64
// ranges at most), then the ranges' sums eight loads ahead, every W-th group of
// eight a wave's. Latency bound: one row of 64 ranges takes 10 us with one wave
// and 6 with four.
template <int QT, int W>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
    __shared__ float part_x[W > 1 ? W : 1][W > 1 ? 256 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), of = wave % W;
    const long long n = (long long)a.n_tok * a.H * a.G;
    const long long row = (long long)blockIdx.x * (4 / W) + wave / W;
    if (row >= n) return;
    const int tok = (int)(row / (a.H * a.G)), head = (int)(row % (a.H * a.G));
    if (tok < a.cu[0] || tok >= a.cu[a.n_seq]) return;   // (W waves of a row alike)
    const bool mine = lane < a.splits;
    const float m = mine ? a.part_ml[2 * (lane * n + row)] : -INFINITY;
    const float part = mine ? a.part_ml[2 * (lane * n + row) + 1] : 0.0f;
    float top = m;
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float w = exp_of(m - (top == -INFINITY ? 0.0f : top));
    float l = w * part;
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float x[4] = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int col = lane + 64 * c;
        if (64 * c >= a.dv) continue;
        const float * from = a.part_o + row * a.dv + (col < a.dv ? col : 0);
        for (int s = 8 * of; s < a.splits; s += 8 * W) {
            float f[8], y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = __shfl(w, (s + j) & 63);
            // (a range that saw nothing has no sums; past the last range w is 0)
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = s + j < a.splits && f[j] != 0.0f ? from[(s + j) * n * a.dv] : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) x[c] += f[j] * y[j];
        }
    }
    if constexpr (W > 1) {
        for (int c = 0; c < 4; c++) part_x[of][lane + 64 * c] = x[c];
        __syncthreads();
        if (of) return;
        for (int c = 0; c < 4; c++)
            for (int v = 1; v < W; v++) x[c] += part_x[v][lane + 64 * c];
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int col = lane + 64 * c;
        if (col >= a.dv) continue;
        const long long at = (long long)tok * a.o_tok + (long long)head * a.o_head + col;
        if constexpr (QT == kF32)
            reinterpret_cast<float *>(a.o)[at] = x[c] * inv;
        else
            reinterpret_cast<unsigned short *>(a.o)[at] = (unsigned short)pack2<QT>(x[c] * inv, x[c] * inv);
    }
    if (a.lse && lane == 0) a.lse[row] = l == 0.0f ? -INFINITY : top + logf(l);
}

template <int QT> bool run_join(const AttnArgs & a, hipStream_t st) {
    const long long rows = (long long)a.n_tok * a.H * a.G;
    // (more than 8 ranges are more than one round of loads; with rows enough to
    // fill the GPU a wave each is faster: 8192 rows of 16 ranges 13 us, 25 with four)
    if (a.splits > 8 && rows <= 1024) return launch(k_attn_join<QT, 4>, dim3((unsigned)rows), dim3(256), st, a);
    return launch(k_attn_join<QT, 1>, dim3((unsigned)((rows + 3) / 4)), dim3(256), st, a);
}

// Row tiles a wave holds: two where there are more than 16 rows, and over a
// Q8_0 cache, whose rows cost more to decode than to multiply, four where
// there are more than 32; at 256 wide heads more than one does not fit the
// registers. Measured, us (8 KV heads of 128, trees; one, two and four tiles):
//   8 sequences of up to 16384 cells, 32 rows   F16 141, 138; F32 311, 295
//   the same, 20 rows                           F16 128, 127; F32 267, 280
//   Q8_0, 16 sequences of up to 32768 cells: 24 rows 454, 414, 460; 36 rows
//     569, 591, 466; 52 rows 797, 631, 471; 64 of up to 8192, 20 rows 491, 429
//   Q8_0, 8 sequences of up to 16384 cells, 32 rows: 146, 195 (one would do
//     better where the call is this small)
//   F32 prompts of 2048 tokens in all, 32 heads: 354, 271
int row_tiles(int type, int d, bool careful, long long rows) {
    if (rows <= 16 || careful || d == 256) return 1;
    return rows > 32 && type == kQ8 ? 4 : 2;
}

// Shape of a cache call's launch (n_seq > 0).
struct CacheShape {
    int rt, tiles, splits, range;
    bool careful;
    int whole;   // waves of rows of k_attn_tiles, 0: k_attn_rows
};
CacheShape cache_shape(const kvc_cache * c, const kvc_cache_attn_args * a, const kvc_window * w) {
    CacheShape s{};
    const int G = a->n_head / c->n_head_kv, es = esize(a->type);
    // a cache's pages are 16-byte aligned: its rows are where a head is whole 16-byte pieces
    s.careful = c->k_type != kQ8 && (!vec_rows(a->q, es) || c->d_k * es % 16 || c->d_v * es % 16);
    const long long rows = (long long)a->max_new * G;
    int max_len = a->max_len < 1 << 30 ? a->max_len : 1 << 30;   // (no sequence has more; sums with it stay in range)
    if (w) {   // (what lies between the first cells and the window is not gone through)
        const long long seen = (long long)w->first + w->last + a->max_new;
        max_len = seen < max_len ? (int)seen : max_len;
    }
    s.rt = row_tiles(c->k_type, head_tile(c->d_k, c->d_v), s.careful, rows);
    // Under a window a call over Q8_0 may be small: row tiles by the keys of all
    // heads. 13 drafts of 32 heads, us with one, two and four tiles a wave, 8 KV
    // heads: 2 sequences that see 512 cells 19, 23 and 33, 2048 23, 24 and 34,
    // 8192 47, 38 and 46; 8 sequences: 20, 25 and 35; 44, 39 and 45; 140, 94 and
    // 90; 16 and 2048: 71, 55 and 64; 32: 53, 53 and 46; 132, 108 and 91; 566, 351
    // and 288. (The keys alone do not tell all: 32 sequences of 512 are given two,
    // where four are faster, because 8 of 2048, as many keys, do better with two.)
    if (w && s.rt > 1 && c->k_type == kQ8) {
        const long long keys = (long long)max_len * a->n_seq * c->n_head_kv;
        s.rt = keys < 1 << 16 ? 1 : keys < 400000 || s.rt == 2 ? 2 : 4;
    }
    // Tiles in LDS from 33 rows on: 8 sequences of up to 20000 F16 cells with a
    // bias, k_attn_rows against two waves of rows: 36 rows 164 and 127 us, 64
    // rows 190 and 133 (24 rows 152 and 121: it would pay earlier); one
    // sequence of 20000: 32 rows 33 both, 36 rows 47 and 34. Four waves of rows
    // from 65 on read a tile for twice as many rows; which is faster goes with
    // the sequences' lengths: 128 rows 157 us against 170 with two, and with
    // other lengths 190 against 183 and 183 against 175; 16 sequences of up to
    // 16384 242 against 260; 64 of up to 4096, 80 rows, 268 against 227.
    if (rows > 32 && !s.careful && c->k_type != kF32 && c->k_type != kQ8 && vec_rows(a->o, es))
        s.whole = rows > 64 && c->d_k <= 128 && c->d_v <= 128 ? 4 : 2;
    const int block_rows = s.whole ? 32 * s.whole : 16 * s.rt;
    const long long tiles = (rows + block_rows - 1) / block_rows;
    // (a block that has no tile of its own goes on with those that the grid has no blocks for)
    const long long room = kMaxBlocks / ((long long)a->n_seq * c->n_head_kv);
    const long long most_tiles = room < 1 ? 1 : room > 65536 ? 65536 : room;
    s.tiles = (int)(tiles < 1 ? 1 : tiles > most_tiles ? most_tiles : tiles);
    // Key ranges: enough blocks to fill the GPU, each with at least 8 tiles of
    // 32 keys. Ranges of the same size in all sequences; four row tiles a wave
    // (one block a CU, and its time goes with its keys) take the same number
    // of ranges of each sequence instead (trees over Q8_0 471 us, 559 with
    // ranges of one size). Measured, us, for 1024 and 4096 blocks: one token of
    // 64 sequences of up to 16384 bf16 cells 559 and 509, Q8_0 642 and 542 (8192:
    // 503 and 497; of 8 sequences 96 and 105); trees of 32 over F16 193 and 319
    // (512: 171), of 13 over Q8_0 469 and 604. For one token of one sequence:
    // 4096 cells in 8, 16 and 32 ranges 17.0, 14.1 and 13.3, 1024 cells in 2, 4
    // and 8 15.2, 12.4 and 11.1. At most 64, the lanes of the join's wave.
    // Under a window every long sequence has as many keys as the others, so that
    // one block a CU is enough and more only cost their beginnings and the join:
    // one token of 8, 32 and 64 sequences that see 2048 keys, for 256, 1024 and
    // 4096 blocks 21, 23 and 23; 48, 55 and 61 us; 64 of 4096 keys 196, 206 and
    // 216; trees of 32 over F16, 32 sequences of 4096 keys 150, 219 and 391. The
    // least keys of a range are two tiles: 2 sequences of 512 keys 12.5 us, 15.2
    // with eight; of 2048 14.9 and 15.3.
    const long long units = (long long)a->n_seq * c->n_head_kv * s.tiles;
    const long long blocks = w ? 256 : s.whole || s.rt == 4 ? 1024 : 4096;
    long long want = (blocks + units - 1) / units, most = max_len / (w ? 64 : 256);
    want = want < most ? want : most;
    if ((long long)a->n_tok * a->n_head > 1 << 24) want = 1;   // (the join's launch: a block a row or four; so many need no ranges)
    s.splits = (int)(want < 1 ? 1 : want > 64 ? 64 : want);
    s.range = s.rt == 4 ? 0 : (max_len + s.splits - 1) / s.splits;
    return s;
}

void set_window(AttnArgs & a, const kvc_window * w) {
    a.first = w->first < 1 << 30 ? w->first : 1 << 30;
    a.last = w->last < 1 << 30 ? w->last : 1 << 30;
}

}  // namespace

int check_window(const kvc_window * w) { return w && (w->first < 0 || w->last < 1) ? -2 : 0; }

int check_cache_attn(const kvc_cache * c, const kvc_cache_attn_args * a) {
    if (int rc = check_cache(c)) return rc;
    if (!a) return -1;
    if (a->n_seq < 0 || a->n_tok < 0 || a->n_head <= 0 || a->max_new < 0 || a->max_len < 0 || a->mask_words < 0 ||
        a->layer < 0 || a->layer >= c->n_layers || a->n_head % c->n_head_kv)
        return -2;
    if ((long long)a->n_tok * a->n_head > kMaxRows || (long long)a->max_new * (a->n_head / c->n_head_kv) > kMaxRows)
        return KV_COMPACT_E_UNSUPPORTED;
    if (c->k_type != c->v_type) return KV_COMPACT_E_UNSUPPORTED;
    if (c->k_type == kQ8 ? a->type != kF16 && a->type != kBF16 : a->type != c->k_type) return KV_COMPACT_E_UNSUPPORTED;
    return 0;
}

int cache_args(const kvc_cache * c, const kvc_cache_attn_args * x, const kvc_window * w, AttnArgs & a) {
    const long long krow = (long long)kv_quant_row_bytes(c->k_type, c->n_head_kv * c->d_k);
    const long long vrow = (long long)kv_quant_row_bytes(c->v_type, c->n_head_kv * c->d_v);
    const long long cells = (long long)c->n_pages * c->page_size;
    if (krow >= 1 << 24 || vrow >= 1 << 24) return KV_COMPACT_E_UNSUPPORTED;
    a = AttnArgs{};
    a.k = RowsAt{static_cast<const char *>(c->K) + x->layer * cells * krow, krow / c->n_head_kv, (unsigned)krow};
    a.v = RowsAt{static_cast<const char *>(c->V) + x->layer * cells * vrow, vrow / c->n_head_kv, (unsigned)vrow};
    a.q = static_cast<const char *>(x->q.data);
    a.o = static_cast<char *>(x->o.data);
    a.q_tok = x->q.ld_tok; a.q_head = x->q.ld_head; a.o_tok = x->o.ld_tok; a.o_head = x->o.ld_head;
    a.lse = x->lse; a.cu = x->cu; a.seqs = x->seqs; a.len = c->len; a.table = c->table;
    a.bias = c->bias ? c->bias + x->layer * cells * c->n_head_kv : nullptr;
    a.mask = reinterpret_cast<const unsigned long long *>(x->mask);
    a.mask_words = x->mask_words; a.n_seq = x->n_seq; a.n_tok = x->n_tok;
    a.H = c->n_head_kv; a.G = x->n_head / c->n_head_kv; a.dk = c->d_k; a.dv = c->d_v;
    a.shift = __builtin_ctz(c->page_size); a.n_pages = c->n_pages; a.max_seqs = c->max_seqs; a.max_pages = c->max_pages;
    a.scale = x->scale != 0.0f ? x->scale : 1.0f / sqrtf((float)c->d_k);
    if (w) set_window(a, w);
    return 0;
}

namespace {

size_t cache_workspace(const kvc_cache * c, const kvc_cache_attn_args * a, const kvc_window * w) {
    if (check_cache_attn(c, a) || check_window(w) || a->n_seq == 0 || a->n_tok == 0) return 0;
    const CacheShape s = cache_shape(c, a, w);
    return s.splits > 1 ? (size_t)s.splits * a->n_tok * a->n_head * (c->d_v + 2) * sizeof(float) : 0;
}

int attn_cache(const kvc_cache * c, const kvc_cache_attn_args * x, const kvc_window * w, void * ws, size_t ws_bytes,
               void * stream) {
    if (int rc = check_cache_attn(c, x)) return rc;
    if (int rc = check_window(w)) return rc;
    if (x->n_seq == 0 || x->n_tok == 0) return 0;
    if (!x->q.data || !x->o.data || !x->cu) return -1;
    const int es = esize(x->type);
    if ((reinterpret_cast<uintptr_t>(x->q.data) | reinterpret_cast<uintptr_t>(x->o.data)) & (es - 1))
        return KV_COMPACT_E_UNSUPPORTED;
    const CacheShape s = cache_shape(c, x, w);
    const size_t need = cache_workspace(c, x, w);
    if (need && !ws) return -1;
    if (need && reinterpret_cast<uintptr_t>(ws) & 15) return KV_COMPACT_E_UNSUPPORTED;
    if (need > ws_bytes) return KVC_E_SCRATCH;
    AttnArgs a;
    if (int rc = cache_args(c, x, w, a)) return rc;
    a.splits = s.splits; a.range = s.range; a.tiles = s.tiles;
    a.part_o = static_cast<float *>(ws);
    a.part_ml = a.part_o + (size_t)s.splits * x->n_tok * x->n_head * c->d_v;
    const long long blocks = (long long)x->n_seq * s.tiles * s.splits * a.H;
    if (blocks > kMaxBlocks) return KV_COMPACT_E_UNSUPPORTED;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    if (!(w ? run_attn_window(a, c->k_type, x->type, s.whole, s.rt, s.careful, blocks, st)
            : run_attn<false>(a, c->k_type, x->type, s.whole, s.rt, s.careful, blocks, st)))
        return KV_COMPACT_E_DEVICE;
    if (s.splits > 1) {
        if (!(x->type == kF32 ? run_join<kF32>(a, st) : x->type == kF16 ? run_join<kF16>(a, st) : run_join<kBF16>(a, st)))
            return KV_COMPACT_E_DEVICE;
    }
    return 0;
}

int attn_prompt(const kvc_prompt_args * x, const kvc_window * w, void * stream) {
    if (!x) return -1;
    if (x->n_seq < 0 || x->n_tok < 0 || x->n_head <= 0 || x->n_head_kv <= 0 || x->d_k <= 0 || x->d_v <= 0 ||
        x->n_head % x->n_head_kv)
        return -2;
    if (int rc = check_window(w)) return rc;
    if ((long long)x->n_tok * x->n_head > kMaxRows || x->d_k > 256 || x->d_v > 256 || (x->type != kF32 && x->type != kF16 && x->type != kBF16))
        return KV_COMPACT_E_UNSUPPORTED;
    if (x->n_seq == 0 || x->n_tok == 0) return 0;
    if (!x->q.data || !x->k.data || !x->v.data || !x->o.data || !x->cu) return -1;
    const int es = esize(x->type), G = x->n_head / x->n_head_kv;
    if ((reinterpret_cast<uintptr_t>(x->q.data) | reinterpret_cast<uintptr_t>(x->k.data) |
         reinterpret_cast<uintptr_t>(x->v.data) | reinterpret_cast<uintptr_t>(x->o.data)) & (es - 1))
        return KV_COMPACT_E_UNSUPPORTED;
    if (x->k.ld_tok < 0 || x->k.ld_tok * es >= 1 << 24 || x->v.ld_tok < 0 || x->v.ld_tok * es >= 1 << 24)
        return KV_COMPACT_E_UNSUPPORTED;
    AttnArgs a{};
    a.k = RowsAt{static_cast<const char *>(x->k.data), x->k.ld_head * es, (unsigned)(x->k.ld_tok * es)};
    a.v = RowsAt{static_cast<const char *>(x->v.data), x->v.ld_head * es, (unsigned)(x->v.ld_tok * es)};
    a.q = static_cast<const char *>(x->q.data);
    a.o = static_cast<char *>(x->o.data);
    a.q_tok = x->q.ld_tok; a.q_head = x->q.ld_head; a.o_tok = x->o.ld_tok; a.o_head = x->o.ld_head;
    a.lse = x->lse; a.cu = x->cu;
    a.n_seq = x->n_seq; a.n_tok = x->n_tok; a.H = x->n_head_kv; a.G = G; a.dk = x->d_k; a.dv = x->d_v;
    a.splits = 1;
    a.scale = x->scale != 0.0f ? x->scale : 1.0f / sqrtf((float)x->d_k);
    const bool careful = !vec_rows(x->q, es) || !vec_rows(x->k, es) || !vec_rows(x->v, es) || x->d_k * es % 16 ||
                         x->d_v * es % 16;
    const bool whole = x->type != kF32 && !careful && vec_rows(x->o, es);
    const int rt = row_tiles(x->type, head_tile(x->d_k, x->d_v), careful, (long long)x->n_tok * G);
    const int block_rows = whole ? 128 : 16 * rt;
    const long long tiles = ((long long)x->n_tok * G + block_rows - 1) / block_rows + x->n_seq;
    if (tiles * a.H > kMaxBlocks) return KV_COMPACT_E_UNSUPPORTED;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    if (w) set_window(a, w);
    return (w ? run_attn_window(a, x->type, x->type, whole ? 4 : 0, rt, careful, tiles * a.H, st)
              : run_attn<false>(a, x->type, x->type, whole ? 4 : 0, rt, careful, tiles * a.H, st))
               ? 0
               : KV_COMPACT_E_DEVICE;
}

}  // namespace

}  // namespace kvc

using namespace kvc;

extern "C" {

size_t kvc_attn_cache_workspace(const kvc_cache * c, const kvc_cache_attn_args * a) { return cache_workspace(c, a, nullptr); }

int kvc_attn_cache(const kvc_cache * c, const kvc_cache_attn_args * a, void * ws, size_t ws_bytes, void * stream) {
    return attn_cache(c, a, nullptr, ws, ws_bytes, stream);
}

size_t kvc_attn_cache_window_workspace(const kvc_cache * c, const kvc_cache_attn_args * a, const kvc_window * w) {
    return w ? cache_workspace(c, a, w) : 0;
}

int kvc_attn_cache_window(const kvc_cache * c, const kvc_cache_attn_args * a, const kvc_window * w, void * ws,
                          size_t ws_bytes, void * stream) {
    return w ? attn_cache(c, a, w, ws, ws_bytes, stream) : -1;
}

int kvc_attn_prompt(const kvc_prompt_args * a, void * stream) { return attn_prompt(a, nullptr, stream); }

int kvc_attn_prompt_window(const kvc_prompt_args * a, const kvc_window * w, void * stream) {
    return w ? attn_prompt(a, w, stream) : -1;
}

}  // extern "C"
