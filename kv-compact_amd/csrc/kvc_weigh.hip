// The softmax weight that tokens give each cell of a cache, added up
// (include/kvc-cache.h, kvc_cache_weigh):
//   w[h][j] = decay w[h][j] + sum over the tokens i that see cell j and the
//             query heads of group h of exp(scale q_i.k_j + bias_j - lse_i).
// With the rows' log-sum-exps at hand there is no running maximum and nothing
// to join: a block keeps its cells' keys and goes over the rows, so that a
// cell's sum is one wave's, in one order, and needs no atomics.
//
// The product is S^T[key][row] = K Q^T as in the attention kernels: a lane
// holds one row of the caller's, so its log-sum-exp is one register, and adds
// up the keys' weights over the row tiles; lanes are summed at the end.
#include "kvc_attn_kernels.h"

#pragma clang fp contract(fast)

namespace kvc {

namespace {

struct WeighArgs {
    AttnArgs a;            // (o and v are not used)
    float * weight;        // this layer's [max_seqs][H][room]
    long long w_seq;       // weights of a sequence (a layer's are max_seqs apart): H * room
    long long room;        // cells of a row of weights
    float decay;
    int tail, fresh;
    int cell_tiles;        // blocks of a sequence's head
};

// What a block of a call works on.
struct Counted {
    Sequence q;
    int seq;         // whose weights
    int tok_from;    // first token that counts
    int old;         // cells before it have gathered weights already
};
__device__ __forceinline__ bool counted_of(const WeighArgs & w, int s, Counted & c) {
    c.q = sequence_of(w.a, s);
    if (c.q.n_new <= 0 || c.q.held == 0) return false;
    c.seq = w.a.seqs ? uniform_load(w.a.seqs + s) : s;
    c.tok_from = w.tail > 0 && w.tail < c.q.n_new ? c.q.n_new - w.tail : 0;
    c.old = w.fresh > c.q.held - c.q.base ? (w.fresh < c.q.held ? c.q.held - w.fresh : 0) : c.q.base;
    return true;
}

// Tokens that may see a cell of cells lo .. hi - 1.
__device__ __forceinline__ void tokens_of(const AttnArgs & a, const Counted & c, int lo, int hi, int & t0, int & t1) {
    t0 = c.tok_from;
    t1 = c.q.n_new;
    if (a.mask) {
        // (the drafts see cells before them by how many of them they see: not looked into)
        if (lo >= a.first && hi <= c.q.base - a.last) t1 = t0;
        return;
    }
    if (lo - c.q.base > t0) t0 = lo - c.q.base;
    if (lo >= a.first && hi - 1 - c.q.base + a.last < t1) t1 = hi - 1 - c.q.base + a.last;
}

__device__ __forceinline__ void add_weight(const WeighArgs & w, const Counted & c, int h, int cell, float sum) {
    if (cell >= c.q.held) return;
    float * at = w.weight + c.seq * w.w_seq + h * w.room + cell;
    *at = (cell < c.old && w.decay != 0.0f ? w.decay * *at : 0.0f) + sum;
}

// Four waves of a block, 32 cells each; rows 16 at a time.
template <int TYPE, int QT, int D, Columns COLS>
__global__ __launch_bounds__(256) void k_weigh_rows(WeighArgs w) {
    using C = RowKernel<TYPE, QT, D, 1, COLS>;
    constexpr bool Q8 = C::Q8;
    __shared__ __align__(16) float k_scale[Q8 ? 4 : 1][Q8 ? C::NB : 1][32];
    const AttnArgs & a = w.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4;
    int u = blockIdx.x;
    const int h = u % a.H;
    u /= a.H;
    const int first_tile = u % w.cell_tiles, s = u / w.cell_tiles;
    Counted c;
    if (!counted_of(w, s, c)) return;
    const Sequence & q = c.q;
    const int page_mask = (1 << a.shift) - 1;

    for (int tile = first_tile; tile * 128LL < q.held; tile += w.cell_tiles) {
        const int cell0 = tile * 128 + 32 * wave;
        if (cell0 >= q.held) continue;
        int t0, t1;
        tokens_of(a, c, cell0, cell0 + 32 < q.held ? cell0 + 32 : q.held, t0, t1);
        float sum[2][4];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) sum[x][i] = 0.0f;
        if (t0 < t1) {
            // keys, and the cells that are not to be read (bad pages; past the end)
            unsigned kr[2][C::NKL][C::WK];
            unsigned there = 0;
            f4 bias[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int cell = cell0 + 16 * x;
                int page = cell < q.held ? uniform_load(q.table + (cell >> a.shift)) : -1;
                if (page >= 0 && page < a.n_pages)
                    there |= (q.held - cell >= 16 ? 0xffffu : (1u << (q.held - cell)) - 1) << (16 * x);
                else
                    page = 0;
                const unsigned row0 = ((unsigned)page << a.shift) + (cell & page_mask);
                const char * p = a.k.base + h * a.k.ld_head + (unsigned long long)row0 * a.k.ld_tok;
                const unsigned row = __umul24(m, a.k.ld_tok);
#pragma unroll
                for (int j = 0; j < C::NKL; j++) {
                    if constexpr (Q8)
                        *reinterpret_cast<u2 *>(kr[x][j]) =
                            COLS == FULL || 32 * j < a.dk ? *reinterpret_cast<const u2_any *>(p + (row + 34 * j + 2 + 8 * g)) : u2{0, 0};
                    else
                        load_cols<C::KV, C::ES, COLS>(p, row, 4 * C::KV * j + C::KV * g, a.dk, kr[x][j]);
                }
                if (a.bias)
                    bias[x] = *reinterpret_cast<const f4 *>(a.bias + (((long long)page * a.H + h) << a.shift) + ((cell + 4 * g) & page_mask));
                if constexpr (Q8) {
                    // scales: lane g * 16 + m takes cell m's blocks g, g + 4, ...
#pragma unroll
                    for (int b = 0; b < (C::NB + 3) / 4; b++) {
                        const int at = 4 * b + g;
                        if (at < C::NB)
                            k_scale[wave][at][16 * x + m] =
                                COLS == FULL || 32 * at < a.dk ? f16_value(*reinterpret_cast<const unsigned short *>(p + row + 34 * at)) : 0.0f;
                    }
                }
            }
            bool hidden = there != ~0u;   // (uniform) a cell that no row sees
            if (a.bias) {
                unsigned off = 0;
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int i = 0; i < 4; i++) off |= bias[x][i] == -INFINITY ? 1u << (16 * x + 4 * g + i) : 0;
                there &= ~off;
                hidden |= __ballot(off != 0) != 0;
            }
            if constexpr (Q8) {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
            const int row_end = t1 * a.G;
            for (int row0 = t0 * a.G; row0 < row_end; row0 += 16) {
                const int row = row0 + m;
                const bool on = row < row_end;
                const int tok = (on ? row : row0) / a.G, head = (on ? row : row0) % a.G;
                u4 qf[C::NK];
                const char * p = a.q + ((long long)(q.tok0 + tok) * a.q_tok + (long long)(h * a.G + head) * a.q_head) * C::ES;
#pragma unroll
                for (int j = 0; j < C::NK; j++) {
                    const int col = 4 * C::KV * j + C::KV * g;
                    if constexpr (Q8) {
                        qf[j] = COLS == FULL || col < a.dk ? *reinterpret_cast<const u4_any *>(p + 2 * col) : u4{0, 0, 0, 0};
                    } else {
                        unsigned x[4];
                        load_cols<C::KV, C::ES, COLS>(p, 0, col, a.dk, x);
                        qf[j] = u4{x[0], x[1], x[2], x[3]};
                    }
                }
                float scale = a.scale, rest = 1.0f;
                if constexpr (Q8 && QT == kBF16) bf16_row_to_f16(qf, a.scale, scale, rest);
                float lse = a.lse[(long long)(q.tok0 + tok) * a.H * a.G + h * a.G + head];
                lse = on && lse != -INFINITY ? lse : INFINITY;   // (a row that saw nothing gives nothing)
                // keys that every row of the tile sees
                const int clear = a.mask ? q.base : q.base + row0 / a.G + 1;
                const int last_tok = (row0 + 15 < row_end ? row0 + 15 : row_end - 1) / a.G;
                const int from = a.mask ? q.base - (q.n_new < a.last ? a.last - q.n_new : 0) : q.base + last_tok + 1 - a.last;
                const bool special = hidden || row0 + 16 > row_end || cell0 + 32 > clear || (cell0 + 32 > a.first && cell0 < from);
                unsigned see = there;
                if (special) {
                    see &= seen32(a, q, tok, cell0) & window32(a, window_from(a, q, tok), cell0);
                    see = on ? see : 0;
                }
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    f4 sc = {0, 0, 0, 0};
                    if constexpr (TYPE == kF32) {
                        f4 part[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) part[e] = f4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < C::NKL; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[x][j][e]),
                                                                               __uint_as_float(qf[j][e]), part[e], 0, 0, 0);
                        sc = (part[0] + part[1]) + (part[2] + part[3]);
                    }
#pragma unroll
                    for (int j = 0; j < (TYPE == kF32 ? 0 : C::NKL); j++) {
                        if constexpr (Q8) {
                            unsigned y[4];
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                y[e] = code_pair(kr[x][j][e >> 1], kr[x][j][e >> 1], e & 1 ? 0x0c030c02u : 0x0c010c00u);
                            const f4 f = *reinterpret_cast<const f4 *>(&k_scale[wave][j][16 * x + 4 * g]);
                            sc += f * mfma16<kF16>(u4{y[0], y[1], y[2], y[3]}, qf[j], f4{0, 0, 0, 0});
                        } else {
                            sc = mfma16<C::MT>(u4{kr[x][j][0], kr[x][j][1], kr[x][j][2], kr[x][j][3]}, qf[j], sc);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // (the difference before log2 e: its rounding goes with the weight's size, not the score's)
                        float v = sc[i] * scale;
                        if constexpr (Q8 && QT == kBF16) v *= rest;
                        if (a.bias) v += bias[x][i];
                        const float p = exp_of(v - lse);
                        sum[x][i] += !special || (see >> (16 * x + 4 * g + i) & 1) ? p : 0.0f;
                    }
                }
            }
        }
        // over the rows; then cell 16 x + 4 g + i is lane 16 g + 4 x + i's
        float mine = 0.0f;
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = sum[x][i];
                for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o);
                mine = m == 4 * x + i ? v : mine;
            }
        if (m < 8) add_weight(w, c, h, cell0 + 16 * (m >> 2) + 4 * g + (m & 3), mine);
    }
}

template <int TYPE, int QT, int D> bool run_weigh(const WeighArgs & w, bool careful, long long blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block(256);
    if constexpr (TYPE != kQ8)
        if (careful) return launch(k_weigh_rows<TYPE, QT, D, ANY>, grid, block, st, w);
    if (w.a.dk == D) return launch(k_weigh_rows<TYPE, QT, D, FULL>, grid, block, st, w);
    return launch(k_weigh_rows<TYPE, QT, D, PART>, grid, block, st, w);
}
template <int TYPE, int QT> bool run_weigh(const WeighArgs & w, bool careful, long long blocks, hipStream_t st) {
    if (w.a.dk <= 64) return run_weigh<TYPE, QT, 64>(w, careful, blocks, st);
    if (w.a.dk <= 128) return run_weigh<TYPE, QT, 128>(w, careful, blocks, st);
    return run_weigh<TYPE, QT, 256>(w, careful, blocks, st);
}

}  // namespace

}  // namespace kvc

using namespace kvc;

extern "C" int kvc_cache_weigh(const kvc_cache * c, const kvc_cache_attn_args * x, const kvc_window * win,
                               const kvc_weigh_args * y, void * stream) {
    if (int rc = check_cache_attn(c, x)) return rc;
    if (!y) return -1;
    if (int rc = check_window(win)) return rc;
    if (y->tail < 0 || y->fresh < 0 || !(y->decay >= 0.0f) || y->decay > 1.0f) return -2;
    if (x->n_seq == 0 || x->n_tok == 0) return 0;
    if (!x->q.data || !x->lse || !x->cu || !y->weight) return -1;
    if ((reinterpret_cast<uintptr_t>(x->q.data) & (esize(x->type) - 1)) || (reinterpret_cast<uintptr_t>(y->weight) & 3))
        return KV_COMPACT_E_UNSUPPORTED;
    const kvc_window all = {0, 1 << 30};
    AttnArgs a;
    if (int rc = cache_args(c, x, win ? win : &all, a)) return rc;
    WeighArgs w{};
    w.room = (long long)c->max_pages * c->page_size;
    w.w_seq = w.room * c->n_head_kv;
    w.weight = y->weight + x->layer * c->max_seqs * w.w_seq;
    w.decay = y->decay;
    w.tail = y->tail;
    w.fresh = y->fresh;
    const int es = esize(x->type);
    const bool careful = c->k_type != kQ8 && (!vec_rows(x->q, es) || c->d_k * es % 16);
    const long long want = (x->max_len + 127LL) / 128, most = kMaxBlocks / ((long long)x->n_seq * c->n_head_kv);
    if (most < 1) return KV_COMPACT_E_UNSUPPORTED;
    w.cell_tiles = (int)(want < 1 ? 1 : want < most ? want : most);
    w.a = a;
    const long long blocks = (long long)x->n_seq * c->n_head_kv * w.cell_tiles;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    bool ok;
    if (c->k_type == kF32) ok = run_weigh<kF32, kF32>(w, careful, blocks, st);
    else if (c->k_type == kF16) ok = run_weigh<kF16, kF16>(w, careful, blocks, st);
    else if (c->k_type == kBF16) ok = run_weigh<kBF16, kBF16>(w, careful, blocks, st);
    else if (x->type == kF16) ok = run_weigh<kQ8, kF16>(w, careful, blocks, st);
    else ok = run_weigh<kQ8, kBF16>(w, careful, blocks, st);
    return ok ? 0 : KV_COMPACT_E_DEVICE;
}
