// The softmax weight that tokens give each cell of a cache, added up
// (include/kvc-cache.h, kvc_cache_weigh):
//   w[h][j] = decay w[h][j] + sum over the tokens i that see cell j and the
//             query heads of group h of exp(scale q_i.k_j + bias_j - lse_i).
// With the rows' log-sum-exps at hand there is no running maximum: a block keeps
// its cells' keys and goes over the rows, so that a cell's sum is one block's, in
// one order, and needs no atomics. It is one wave's, but in the forms for few
// blocks, where two waves (k_weigh_tiles) or four (k_weigh_rows) share out the
// rows and join their parts in LDS.
//
// The product is S^T[key][row] = K Q^T as in the attention kernels: a lane
// holds one row of the caller's, so its log-sum-exp is one register, and adds
// up the keys' weights over the row tiles; lanes are summed at the end.
#include "kvc_attn_kernels.h"

#include <type_traits>
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
    int range;             // k_weigh_few, k_weigh_ring: groups of 32 or 64 cells of each, at least
    float to_log2;         // k_weigh_tiles: scale times log2 e, rounded
    float lse_log2[2];     // the same of a log-sum-exp: to_log2 / scale in two parts
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

// Rows whose log-sum-exp is -inf give nothing, whatever their queries hold: cells
// are hidden from them as they are by a mask. With few rows a block knows whether
// it has such ones. The kernels for many rows take a log-sum-exp of +inf for them,
// which gives 0 but for scores that are NaN or +inf, and go through a tile of cells
// once more, masks everywhere, where a sum is NaN. (A look at each tile of rows:
// 4096 tokens 156 us, 151 so; over Q8_0 460 and 447.)
// Rows behind the last repeat it, with +inf; one that saw nothing keeps its -inf.
__device__ __forceinline__ float row_log_sum(float lse, bool on) { return on || lse == -INFINITY ? lse : INFINITY; }

// (what the first of two passes derives from x is not kept in registers for the second)
__device__ __forceinline__ int opaque(int x) {
    x = __builtin_amdgcn_readfirstlane(x);
    asm volatile("" : "+s"(x));
    return x;
}

// Whether a sum of the block's is NaN (seen: a word a wave; all waves call).
template <int N, int WAVES> __device__ __forceinline__ bool any_nan(const float (&sum)[N], int (&seen)[WAVES]) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; i++) nan |= sum[i] != sum[i];
    nan = __ballot(nan) != 0;
    if ((threadIdx.x & 63) == 0) seen[threadIdx.x >> 6] = nan;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) any |= seen[i];
    return __builtin_amdgcn_readfirstlane(any) != 0;
}

__device__ __forceinline__ void add_weight(const WeighArgs & w, const Counted & c, int h, int cell, float sum) {
    if (cell >= c.q.held) return;
    float * at = w.weight + c.seq * w.w_seq + h * w.room + cell;
    *at = (cell < c.old && w.decay != 0.0f ? w.decay * *at : 0.0f) + sum;
}

// Blocks of 128 cells below which k_weigh_rows splits rows over waves. One prompt,
// 8 KV heads of 128, 32 heads, whole and split, us: F32 1024 tokens 401 and 165,
// 4096 (256 blocks) 1621 and 1086, 8192 3972 and 4244; over Q8_0 1024 tokens 184
// and 100, 4096 718 and 444, 8192 1526 and 1473, 16384 3298 and 5638.
constexpr int kSplit = 512;
constexpr int kFewRows16 = 8, kFewRows32 = 4;   // row tiles of 16 that stay, of 16-bit and F32 rows

// Sum over the 16 lanes of a row of v[m % 8] (lanes m and m ^ 8 alike): each
// step hands half of the values to the lane across.
__device__ __forceinline__ float sum_of_16(float (&v)[8], int m) {
    auto dpp = [](float x, auto ctrl) {
        constexpr int c = decltype(ctrl)::value;
        return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), c, 0xf, 0xf, true));
    };
    using half_mirror = std::integral_constant<int, 0x141>;
    using xor2 = std::integral_constant<int, 0x4e>;
    using xor1 = std::integral_constant<int, 0xb1>;
    using ror8 = std::integral_constant<int, 0x128>;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float mine = m & 4 ? v[4 + i] : v[i], theirs = m & 4 ? v[i] : v[4 + i];
        v[i] = mine + dpp(theirs, half_mirror{});
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float mine = m & 2 ? v[2 + i] : v[i], theirs = m & 2 ? v[i] : v[2 + i];
        v[i] = mine + dpp(theirs, xor2{});
    }
    const float mine = m & 1 ? v[1] : v[0], theirs = m & 1 ? v[0] : v[1];
    const float x = mine + dpp(theirs, xor1{});
    return x + dpp(x, ror8{});
}

// Many rows of F32 or over Q8_0 keys, and rows of any alignment: four waves of a
// block keep 32 cells' keys each in registers (Q8_0 ones decoded), and rows come
// 16 RT at a time through LDS, as the fragments they are, for all four. SPLIT,
// for few blocks: the four have the same 32 cells and every fourth row tile each.
// Bound by what a row tile issues in turn (F32: 32 products in a chain of four
// sums): 4096 tokens of 32 heads of 128, F32 1.01 ms, 68 TFLOP/s (a large product:
// 152); over Q8_0 0.45 ms, 154 TFLOP/s, 16384 tokens 3.3 ms, 332 TFLOP/s. 128-wide
// heads have registers for three waves a SIMD (F32 1.09 ms and Q8_0 0.49 ms with
// the two that the compiler takes by itself), F32 heads from 65 to 127 do not.
template <int TYPE, int QT, int D, int RT, Columns COLS, bool SPLIT>
__global__ __launch_bounds__(256, D == 128 && !(TYPE == kF32 && COLS == PART) ? 3 : 1) void k_weigh_rows(WeighArgs w) {
    constexpr int CELLS = SPLIT ? 32 : 128;
    using C = RowKernel<TYPE, QT, D, 1, COLS>;
    constexpr bool Q8 = C::Q8;
    __shared__ __align__(16) u4 rows_q[RT][C::NK][64];
    __shared__ float rows_scale[Q8 ? RT : 1][2][16];
    __shared__ float rows_lse[RT][2][16];   // as subtracted, and as given
    __shared__ int sums_nan[4];
    __shared__ __align__(16) float k_scale[Q8 ? 4 : 1][Q8 ? C::NB : 1][32];
    __shared__ float join[SPLIT ? 4 : 1][32];
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

    for (int tile = first_tile; (long long)tile * CELLS < q.held; tile += w.cell_tiles) {
        __syncthreads();   // (what waves left each other of the last tile is read; this one may have no rows, and no barrier of theirs)
        const int block0 = tile * CELLS, cell0 = SPLIT ? block0 : block0 + 32 * wave;
        int t0, t1;   // the block's tokens (a wave past the sequence's end has none that see its cells)
        tokens_of(a, c, block0, block0 + CELLS < q.held ? block0 + CELLS : q.held, t0, t1);
        float sum[8];
        // keys, and the cells that rows may see (not those of bad pages or past the end)
        unsigned kr[2][C::NKL][Q8 ? 4 : C::WK];
        f4 ks[Q8 ? 2 : 1][Q8 ? C::NB : 1];
        unsigned there = 0;
        f4 bias[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
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
                if constexpr (Q8) {
                    const u2 y = COLS == FULL || 32 * j < a.dk ? *reinterpret_cast<const u2_any *>(p + (row + 34 * j + 2 + 8 * g)) : u2{0, 0};
#pragma unroll
                    for (int e = 0; e < 4; e++) kr[x][j][e] = code_pair(y[e >> 1], y[e >> 1], e & 1 ? 0x0c030c02u : 0x0c010c00u);
                } else {
                    load_cols<C::KV, C::ES, COLS>(p, row, 4 * C::KV * j + C::KV * g, a.dk, kr[x][j]);
                }
            }
            if (a.bias)
                bias[x] = *reinterpret_cast<const f4 *>(a.bias + (((long long)page * a.H + h) << a.shift) + ((cell + 4 * g) & page_mask));
            if constexpr (Q8) {
                // lane g * 16 + m: blocks g, g + 4, ... of cell m, on their way to the lanes that hold its sums
#pragma unroll
                for (int b = 0; b < (C::NB + 3) / 4; b++) {
                    const int at = 4 * b + g;
                    if (at < C::NB)
                        k_scale[wave][at][16 * x + m] =
                            COLS == FULL || 32 * at < a.dk ? f16_value(*reinterpret_cast<const unsigned short *>(p + row + 34 * at)) : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (bias[x][i] == -INFINITY) there &= ~(1u << (16 * x + 4 * g + i));
        }
        if constexpr (Q8) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int j = 0; j < C::NB; j++) ks[x][j] = *reinterpret_cast<const f4 *>(&k_scale[wave][j][16 * x + 4 * g]);
        }
        const int row_end = t1 * a.G;
        for (bool again = false;; again = true) {
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] = 0.0f;
            for (int turn = opaque(t0) * a.G; turn < row_end; turn += 16 * RT) {
                const int rows = row_end - turn < 16 * RT ? row_end - turn : 16 * RT, row_tiles = (rows + 15) >> 4;
                __syncthreads();   // (the rows before are read)
                for (int r = wave; r < row_tiles; r += 4) {
                    const bool on = 16 * r + m < rows;
                    const int row = turn + (on ? 16 * r + m : rows - 1), tok = row / a.G, head = row % a.G;
                    const char * p = a.q + ((long long)(q.tok0 + tok) * a.q_tok + (long long)(h * a.G + head) * a.q_head) * C::ES;
                    u4 qf[C::NK];
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
#pragma unroll
                    for (int j = 0; j < C::NK; j++) rows_q[r][j][lane] = qf[j];
                    if (g == 0) {
                        const float lse = a.lse[(long long)(q.tok0 + tok) * a.H * a.G + h * a.G + head];
                        rows_lse[r][0][m] = on && lse != -INFINITY ? lse : INFINITY;
                        rows_lse[r][1][m] = lse;
                        if constexpr (Q8) {
                            rows_scale[r][0][m] = scale;
                            rows_scale[r][1][m] = rest;
                        }
                    }
                }
                __syncthreads();
                if (cell0 >= q.held) continue;
                for (int r = SPLIT ? wave : 0; r < row_tiles; r += SPLIT ? 4 : 1) {
                    const int row0 = turn + 16 * r, last_row = row0 + 15 < row_end ? row0 + 15 : row_end - 1;
                    const int first_tok = row0 / a.G, last_tok = last_row / a.G;
                    if (!a.mask && cell0 > q.base + last_tok) continue;   // (no row of the tile sees the cells)
                    u4 qf[C::NK];
#pragma unroll
                    for (int j = 0; j < C::NK; j++) qf[j] = rows_q[r][j][lane];
                    const float lse = rows_lse[r][0][m], scale = Q8 ? rows_scale[r][0][m] : a.scale, rest = Q8 ? rows_scale[r][1][m] : 1.0f;
                    const int clear = a.mask ? q.base : q.base + first_tok + 1;
                    const int from = a.mask ? q.base - (q.n_new < a.last ? a.last - q.n_new : 0) : q.base + last_tok + 1 - a.last;
                    const bool special = cell0 + 32 > clear || (cell0 + 32 > a.first && cell0 < from) || again;
                    unsigned see = ~0u;
                    if (special) {
                        const int tok = (row0 + m < row_end ? row0 + m : row_end - 1) / a.G;
                        see = rows_lse[r][1][m] == -INFINITY ? 0 : seen32(a, q, tok, cell0) & window32(a, window_from(a, q, tok), cell0);
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
                            const u4 kf = {kr[x][j][0], kr[x][j][1], kr[x][j][2], kr[x][j][3]};
                            if constexpr (Q8)
                                sc += ks[x][j] * mfma16<kF16>(kf, qf[j], f4{0, 0, 0, 0});
                            else
                                sc = mfma16<C::MT>(kf, qf[j], sc);
                        }
                        float p[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            // (the difference before log2 e: its rounding goes with the weight's size, not the score's)
                            float v = sc[i];
                            if constexpr (Q8 && QT == kBF16) v *= rest;
                            p[i] = exp_of(__builtin_fmaf(v, scale, bias[x][i]) - lse);
                        }
                        if (special) {
#pragma unroll
                            for (int i = 0; i < 4; i++) p[i] = see >> (16 * x + 4 * g + i) & 1 ? p[i] : 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) sum[4 * x + i] += p[i];
                    }
                }
            }
            if (again) break;
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] = there >> (16 * (i >> 2) + 4 * g + (i & 3)) & 1 ? sum[i] : 0.0f;
            if (!any_nan(sum, sums_nan)) break;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] = there >> (16 * (i >> 2) + 4 * g + (i & 3)) & 1 ? sum[i] : 0.0f;
        float all = sum_of_16(sum, m);
        if constexpr (SPLIT) {
            const int at = 16 * (m >> 2 & 1) + 4 * g + (m & 3);
            if (m < 8) join[wave][at] = all;
            __syncthreads();
            all = (join[0][at] + join[1][at]) + (join[2][at] + join[3][at]);
            if (wave) continue;
        }
        if (m < 8) add_weight(w, c, h, cell0 + 16 * (m >> 2) + 4 * g + (m & 3), all);
    }
}

// Few rows: 16 RT of them stay (RT = 1: in registers, more in LDS as the
// fragments they are), and a block's waves go through a range of cells, 32 at a
// time, the next ones' keys, biases and old weights on their way meanwhile.
// (More rows than the launch was told of come in turns of as many; a cell's
// weight is then added to by the lane that wrote it.)
// The last 32 tokens of 32 heads over eight F16 caches of up to 20000 cells, 8 x
// 128 with a bias: 57 to 59 us, 3.7 TB/s; its reads with one row tile of eight 49
// us. (Asking once a group of cells, not for each 16 rows, whether some row sees
// less: 62 us, 71 before, for two divisions and a branch beside eight products.)
// One token of 64 sequences of up to 16384 Q8_0 cells: 242 us.
template <int TYPE, int QT, int D, int RT, Columns COLS>
__global__ __launch_bounds__(256) void k_weigh_few(WeighArgs w) {
    using C = RowKernel<TYPE, QT, D, 1, COLS>;
    constexpr bool Q8 = C::Q8;
    constexpr int NS = Q8 ? (C::NB + 3) / 4 : 1;              // scales a lane loads of a group of 16 cells
    constexpr bool AHEAD = 2 * C::NKL * C::WK <= 64;          // the next keys have registers of their own
    __shared__ __align__(16) u4 rows_q[RT > 1 ? RT : 1][RT > 1 ? C::NK : 1][64];
    __shared__ float rows_scale[RT > 1 && Q8 ? RT : 1][2][16];
    __shared__ float rows_lse[RT > 1 ? RT : 1][16];
    __shared__ int rows_nothing[4];
    __shared__ __align__(16) float k_scale[Q8 ? 4 : 1][Q8 ? C::NB : 1][32];
    const AttnArgs & a = w.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4;
    int u = blockIdx.x;
    const int h = u % a.H;
    u /= a.H;
    const int split = u % w.cell_tiles, s = u / w.cell_tiles;
    Counted c;
    if (!counted_of(w, s, c)) return;
    const Sequence & q = c.q;
    const int page_mask = (1 << a.shift) - 1;
    const int all_rows = (q.n_new - c.tok_from) * a.G;
    const int n_groups = (q.held + 31) >> 5;
    const int even = (n_groups + w.cell_tiles - 1) / w.cell_tiles, per = even > w.range ? even : w.range;
    const int g_lo = split * per, g_hi = g_lo + per < n_groups ? g_lo + per : n_groups;
    if (g_lo >= g_hi) return;

    // row `row` of a turn's (those past the last repeat it, and give nothing)
    int row_lo = 0, rows = 0;
    auto load_row = [&](int row, u4 (&x)[C::NK], float & lse, float & scale, float & rest) {
        const bool on = row < rows;
        row = row_lo + (on ? row : rows - 1);
        const int tok = c.tok_from + row / a.G, head = row % a.G;
        const char * p = a.q + ((long long)(q.tok0 + tok) * a.q_tok + (long long)(h * a.G + head) * a.q_head) * C::ES;
#pragma unroll
        for (int j = 0; j < C::NK; j++) {
            const int col = 4 * C::KV * j + C::KV * g;
            if constexpr (Q8) {
                x[j] = COLS == FULL || col < a.dk ? *reinterpret_cast<const u4_any *>(p + 2 * col) : u4{0, 0, 0, 0};
            } else {
                unsigned y[4];
                load_cols<C::KV, C::ES, COLS>(p, 0, col, a.dk, y);
                x[j] = u4{y[0], y[1], y[2], y[3]};
            }
        }
        scale = a.scale;
        rest = 1.0f;
        if constexpr (Q8 && QT == kBF16) bf16_row_to_f16(x, a.scale, scale, rest);
        lse = a.lse[(long long)(q.tok0 + tok) * a.H * a.G + h * a.G + head];
        lse = row_log_sum(lse, on);
    };

    unsigned kr[2][C::NKL][C::WK], next_kr[AHEAD ? 2 : 1][AHEAD ? C::NKL : 1][C::WK];
    f4 bias[2], next_bias[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    float old = 0.0f, next_old = 0.0f;
    unsigned short scales[2][NS];
    int page[2], next_page[2];
    const int out_at = 16 * (m >> 2 & 1) + 4 * g + (m & 3);   // the cell of a group whose sum this lane (m < 8) gets
    auto pages_of = [&](int t, int (&pg)[2]) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int cell = 32 * t + 16 * x;
            pg[x] = t < g_hi && cell < q.held ? uniform_load(q.table + (cell >> a.shift)) : -1;
        }
    };
    auto good = [&](int pg) { return pg >= 0 && pg < a.n_pages; };
    auto load_keys = [&](int t, const int (&pg)[2], auto & to) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int cell = 32 * t + 16 * x, pg_x = good(pg[x]) ? pg[x] : 0;
            const unsigned row0 = ((unsigned)pg_x << a.shift) + (cell & page_mask);
            const char * p = a.k.base + h * a.k.ld_head + (unsigned long long)row0 * a.k.ld_tok;
            const unsigned row = __umul24(m, a.k.ld_tok);
#pragma unroll
            for (int j = 0; j < C::NKL; j++) {
                if constexpr (Q8)
                    *reinterpret_cast<u2 *>(to[x][j]) =
                        COLS == FULL || 32 * j < a.dk ? *reinterpret_cast<const u2_any *>(p + (row + 34 * j + 2 + 8 * g)) : u2{0, 0};
                else
                    load_cols<C::KV, C::ES, COLS>(p, row, 4 * C::KV * j + C::KV * g, a.dk, to[x][j]);
            }
            if constexpr (Q8) {
                // lane g * 16 + m: blocks g, g + 4, ... of cell m
#pragma unroll
                for (int b = 0; b < NS; b++) {
                    const int at = 4 * b + g;
                    scales[x][b] = at < C::NB && (COLS == FULL || 32 * at < a.dk) ? *reinterpret_cast<const unsigned short *>(p + row + 34 * at) : 0;
                }
            }
            if (a.bias) next_bias[x] = *reinterpret_cast<const f4 *>(a.bias + (((long long)pg_x * a.H + h) << a.shift) + ((cell + 4 * g) & page_mask));
        }
        const int cell = 32 * t + out_at;
        next_old = 0.0f;
        if (m < 8 && (row_lo ? cell < q.held : w.decay != 0.0f && cell < c.old)) next_old = w.weight[c.seq * w.w_seq + h * w.room + cell];
    };

    for (; row_lo < all_rows; row_lo += 16 * RT) {
        rows = all_rows - row_lo < 16 * RT ? all_rows - row_lo : 16 * RT;
        const int row_tiles = (rows + 15) >> 4, t0 = g_lo + wave;
        // cells that every row of the turn sees: those before clear, first or not before from
        const int first_tok = c.tok_from + row_lo / a.G, last_tok = c.tok_from + (row_lo + rows - 1) / a.G;
        const int clear = a.mask ? q.base : q.base + first_tok + 1;
        const int from = a.mask ? q.base - (q.n_new < a.last ? a.last - q.n_new : 0) : q.base + last_tok + 1 - a.last;
        pages_of(t0, page);
        pages_of(t0 + 4, next_page);
        if constexpr (AHEAD)
            if (t0 < g_hi) load_keys(t0, page, next_kr);
        u4 q0[C::NK];
        float lse0 = 0.0f, scale0 = 0.0f, rest0 = 0.0f;
        bool nothing = false;   // a row with a log-sum-exp of -inf
        if constexpr (RT == 1) {
            load_row(m, q0, lse0, scale0, rest0);
            nothing = __ballot(lse0 == -INFINITY) != 0;
        } else {
            if (row_lo) __syncthreads();   // (the rows before are read)
            for (int r = wave; r < row_tiles; r += 4) {
                load_row(16 * r + m, q0, lse0, scale0, rest0);
                nothing |= lse0 == -INFINITY;
#pragma unroll
                for (int j = 0; j < C::NK; j++) rows_q[r][j][lane] = q0[j];
                if (g == 0) {
                    rows_lse[r][m] = lse0;
                    if constexpr (Q8) {
                        rows_scale[r][0][m] = scale0;
                        rows_scale[r][1][m] = rest0;
                    }
                }
            }
            nothing = __ballot(nothing) != 0;
            if (lane == 0) rows_nothing[wave] = nothing;
            __syncthreads();
            nothing = __builtin_amdgcn_readfirstlane(rows_nothing[0] | rows_nothing[1] | rows_nothing[2] | rows_nothing[3]);
        }

        for (int t = t0; t < g_hi; t += 4) {
            const int cell0 = 32 * t;
            if constexpr (AHEAD) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int j = 0; j < C::NKL; j++)
#pragma unroll
                        for (int y = 0; y < C::WK; y++) kr[x][j][y] = next_kr[x][j][y];
            } else {
                load_keys(t, page, kr);
            }
            unsigned there = 0;   // cells that rows may see
#pragma unroll
            for (int x = 0; x < 2; x++) {
                bias[x] = next_bias[x];
                const int left = q.held - cell0 - 16 * x;
                if (good(page[x])) there |= (left >= 16 ? 0xffffu : left <= 0 ? 0u : (1u << left) - 1) << (16 * x);
                if (a.bias)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (bias[x][i] == -INFINITY) there &= ~(1u << (16 * x + 4 * g + i));
                if constexpr (Q8)
#pragma unroll
                    for (int b = 0; b < NS; b++)
                        if (4 * b + g < C::NB) k_scale[wave][4 * b + g][16 * x + m] = f16_value(scales[x][b]);
            }
            old = next_old;
            if constexpr (AHEAD) {
                if (t + 4 < g_hi) load_keys(t + 4, next_page, next_kr);
            }
#pragma unroll
            for (int x = 0; x < 2; x++) page[x] = next_page[x];
            pages_of(t + 8, next_page);
            if constexpr (Q8) {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
            float sum[8];
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] = 0.0f;
            auto sixteen = [&](int r, auto hides) {   // (a constant where there are tiles)
                const int row0 = 16 * r;
                u4 qr[C::NK];
                float lse = lse0, scale = scale0, rest = rest0;
                if constexpr (RT > 1) {
#pragma unroll
                    for (int j = 0; j < C::NK; j++) qr[j] = rows_q[r][j][lane];
                    lse = rows_lse[r][m];
                    scale = a.scale;
                    if constexpr (Q8) {
                        scale = rows_scale[r][0][m];
                        rest = rows_scale[r][1][m];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < C::NK; j++) qr[j] = q0[j];
                }
                unsigned see = ~0u;
                if (hides) {
                    const int row = row0 + m < rows ? row0 + m : rows - 1, tok = c.tok_from + (row_lo + row) / a.G;
                    see = lse == -INFINITY ? 0 : seen32(a, q, tok, cell0) & window32(a, window_from(a, q, tok), cell0);
                }
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    f4 sc = {0, 0, 0, 0};
                    float p[4];
                    if constexpr (TYPE == kF32) {
                        f4 part[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) part[e] = f4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < C::NKL; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[x][j][e]),
                                                                               __uint_as_float(qr[j][e]), part[e], 0, 0, 0);
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
                            sc += f * mfma16<kF16>(u4{y[0], y[1], y[2], y[3]}, qr[j], f4{0, 0, 0, 0});
                        } else {
                            sc = mfma16<C::MT>(u4{kr[x][j][0], kr[x][j][1], kr[x][j][2], kr[x][j][3]}, qr[j], sc);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // (the difference before log2 e: its rounding goes with the weight's size, not the score's)
                        float v = sc[i];
                        if constexpr (Q8 && QT == kBF16) v *= rest;
                        p[i] = exp_of(__builtin_fmaf(v, scale, bias[x][i]) - lse);
                    }
                    if (hides) {
#pragma unroll
                        for (int i = 0; i < 4; i++) p[i] = see >> (16 * x + 4 * g + i) & 1 ? p[i] : 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) sum[4 * x + i] += p[i];
                }
            };
            const bool hides = cell0 + 32 > clear || (cell0 + 32 > a.first && cell0 < from) || nothing;
            if constexpr (RT == 1) {
                sixteen(0, hides);
            } else if (hides) {
                for (int r = 0; r < row_tiles; r++) sixteen(r, std::true_type{});
            } else {
                for (int r = 0; r < row_tiles; r++) sixteen(r, std::false_type{});
            }
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] = there >> (16 * (i >> 2) + 4 * g + (i & 3)) & 1 ? sum[i] : 0.0f;
            const float all = sum_of_16(sum, m);
            const int cell = cell0 + out_at;
            if (m < 8 && cell < q.held) w.weight[c.seq * w.w_seq + h * w.room + cell] = (row_lo ? old : w.decay * old) + all;
        }
    }
}

template <int TYPE, int QT, int D, int RT> bool run_weigh_few(const WeighArgs & w, bool careful, long long blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block(256);
    if constexpr (TYPE != kQ8)
        if (careful) return launch(k_weigh_few<TYPE, QT, D, RT, ANY>, grid, block, st, w);
    if (w.a.dk == D) return launch(k_weigh_few<TYPE, QT, D, RT, FULL>, grid, block, st, w);
    return launch(k_weigh_few<TYPE, QT, D, RT, PART>, grid, block, st, w);
}
template <int TYPE, int QT, int RT> bool run_weigh_few(const WeighArgs & w, bool careful, long long blocks, hipStream_t st) {
    if (w.a.dk <= 64) return run_weigh_few<TYPE, QT, 64, RT>(w, careful, blocks, st);
    if (w.a.dk <= 128) return run_weigh_few<TYPE, QT, 128, RT>(w, careful, blocks, st);
    return run_weigh_few<TYPE, QT, 256, RT>(w, careful, blocks, st);
}
template <int TYPE, int QT> bool run_weigh_few(const WeighArgs & w, long long rows, bool careful, long long blocks, hipStream_t st) {
    if (rows <= 16) return run_weigh_few<TYPE, QT, 1>(w, careful, blocks, st);
    return run_weigh_few<TYPE, QT, TYPE == kF32 ? kFewRows32 : kFewRows16>(w, careful, blocks, st);
}

// (4 bytes a lane, lanes' to side by side)
__device__ __forceinline__ void load_lds4(const char * from, unsigned offset, char * to) {
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)to;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(from), "s"(at) : "m0", "memory");
}

// Up to 16 rows of aligned types: bound by the read of the keys. Each wave has a
// ring of its own in LDS, 16 cells a place, filled by direct loads of 1 KB (whole
// rows of a head; loads to registers in the products' layout take a row in four
// pieces of 64 bytes), and no barrier. It goes through 64 cells at a time: their
// biases and old weights are one load each, their sums one store.
// One token of 32 heads over 64 sequences of up to 16384 bf16 cells, 8 x 128: 262
// us, 5.0 TB/s (a plain read: 6.8; keys in registers, a group of 32 cells ahead:
// 290 us). One sequence of 20000 cells: 12.7 us.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void k_weigh_ring(WeighArgs w) {
    using C = RowKernel<TYPE, TYPE, D, 1, FULL>;
    constexpr int ROWB = D * C::ES, PR = ROWB / 16;                  // bytes and pieces of a row
    constexpr int RPL = 1024 / ROWB, NL = 16 / RPL;                   // rows of a direct load; loads of 16 cells
    constexpr int BUFS = ROWB <= 128 ? 8 : ROWB <= 512 ? 4 : 2, AHEAD = BUFS - 1;   // (two blocks a CU, one from 512 bytes on)
    constexpr int SWAP = PR < 16 ? PR - 1 : 15;                       // bits of a cell's number that its pieces are exchanged by
    constexpr int GB = BUFS / 4 + 2;                                  // groups whose biases and weights are on their way or in use
    __shared__ __align__(16) char ring[4][BUFS][16 * ROWB];
    __shared__ __align__(16) float cell_bias[4][GB][64], cell_old[4][GB][64];
    const AttnArgs & a = w.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4;
    int u = blockIdx.x;
    const int h = u % a.H;
    u /= a.H;
    const int split = u % w.cell_tiles, s = u / w.cell_tiles;
    Counted c;
    if (!counted_of(w, s, c)) return;
    const Sequence & q = c.q;
    const int page_mask = (1 << a.shift) - 1;
    const int all_rows = (q.n_new - c.tok_from) * a.G;
    const int n_groups = (q.held + 63) >> 6;
    const int even = (n_groups + w.cell_tiles - 1) / w.cell_tiles, per = even > w.range ? even : w.range;
    const int g_lo = split * per, g_hi = g_lo + per < n_groups ? g_lo + per : n_groups;
    const int groups = (g_hi - g_lo - wave + 3) >> 2;                 // of this wave: g_lo + wave, every fourth
    if (g_lo + wave >= g_hi) return;
    const int out_at = 16 * (m >> 2) + 4 * g + (m & 3);               // the cell of 64 whose sum this lane gets

    unsigned load_off[NL];
    bool load_on[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int row = i * RPL + lane / PR, piece = (lane % PR) ^ (row & SWAP);
        load_off[i] = __umul24(row, a.k.ld_tok) + 16 * piece;
        load_on[i] = piece * C::KV < a.dk;
    }
    if (a.dk < D) {
        for (int i = lane; i < BUFS * 16 * PR; i += 64) reinterpret_cast<u4 *>(ring[wave])[i] = u4{0, 0, 0, 0};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (direct loads take another way to LDS)
    }

    for (int row_lo = 0; row_lo < all_rows; row_lo += 16) {           // (more rows than the launch was told of: in turns)
        const int rows = all_rows - row_lo < 16 ? all_rows - row_lo : 16;
        // places of 16 cells in this wave's order
        const int places = 4 * groups;
        auto cell_of = [&](int t) { return 64 * (g_lo + wave + 4 * (t >> 2)) + 16 * (t & 3); };
        auto page_of = [&](int t) {
            const int cell = cell_of(t);
            return t < places && cell < q.held ? uniform_load(q.table + (cell >> a.shift)) : -1;
        };
        int load_t = 0, load_buf = 0, load_page = page_of(0);
        // (past the last place: page 0 again, for the count of loads; at least NL of each place)
        auto fill = [&] {
            const int cell = cell_of(load_t), page = load_page >= 0 && load_page < a.n_pages ? load_page : 0;
            const unsigned row = ((unsigned)page << a.shift) + (cell & page_mask);
            const char * from = a.k.base + h * a.k.ld_head + (unsigned long long)row * a.k.ld_tok;
#pragma unroll
            for (int i = 0; i < NL; i++)
                if (load_on[i]) load_lds16(from, load_off[i], &ring[wave][load_buf][i * 1024]);
            if ((load_t & 3) == 0 && load_t < places) {
                // biases (-inf: not there) and old weights of 64 cells, a lane each
                const int at = cell + lane, b = (load_t >> 2) % GB;
                // (by scalar loads: the wait for a vector one would be one for the keys on their way)
                const int pages[4] = {load_page, page_of(load_t + 1), page_of(load_t + 2), page_of(load_t + 3)};
                int pg = lane < 32 ? (lane < 16 ? pages[0] : pages[1]) : lane < 48 ? pages[2] : pages[3];
                if (at >= q.held) pg = -1;
                const char * from_b = reinterpret_cast<const char *>(&hidden_word);
                if (pg >= 0 && pg < a.n_pages)
                    from_b = a.bias ? reinterpret_cast<const char *>(a.bias + (((long long)pg * a.H + h) << a.shift) + (at & page_mask))
                                    : reinterpret_cast<const char *>(&zero_word);
                load_lds4(from_b, reinterpret_cast<char *>(cell_bias[wave][b]));
                const bool kept = row_lo ? at < q.held : w.decay != 0.0f && at < c.old;
                load_lds4(kept ? reinterpret_cast<const char *>(w.weight + c.seq * w.w_seq + h * w.room + at)
                               : reinterpret_cast<const char *>(&zero_word),
                          reinterpret_cast<char *>(cell_old[wave][b]));
            }
            load_t++;
            load_buf = load_buf + 1 < BUFS ? load_buf + 1 : 0;
            load_page = page_of(load_t);
        };
        // this lane's row (those past the last repeat it, and give nothing)
        const bool on = m < rows;
        const int row = row_lo + (on ? m : rows - 1), tok = c.tok_from + row / a.G, head = row % a.G;
        u4 qf[C::NK];
        {
            const char * p = a.q + ((long long)(q.tok0 + tok) * a.q_tok + (long long)(h * a.G + head) * a.q_head) * C::ES;
#pragma unroll
            for (int j = 0; j < C::NK; j++) {
                const int col = 4 * C::KV * j + C::KV * g;
                qf[j] = col < a.dk ? *reinterpret_cast<const u4 *>(p + col * C::ES) : u4{0, 0, 0, 0};
            }
        }
        float lse = a.lse[(long long)(q.tok0 + tok) * a.H * a.G + h * a.G + head];
        lse = row_log_sum(lse, on);
        const int first_tok = c.tok_from + row_lo / a.G, last_tok = c.tok_from + (row_lo + rows - 1) / a.G;
        const int clear = a.mask ? q.base : q.base + first_tok + 1;
        const int cut = a.mask ? q.base - (q.n_new < a.last ? a.last - q.n_new : 0) : q.base + last_tok + 1 - a.last;
        const int from = window_from(a, q, tok);
        // (waited for here: a wait in the loop would be one for the keys on their way too)
#pragma unroll
        for (int j = 0; j < C::NK; j++) asm volatile("" : "+v"(qf[j]));
        asm volatile("" : "+v"(lse));
        const bool nothing = __ballot(lse == -INFINITY) != 0;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) fill();

        float mine = 0.0f;
        int buf = 0;
        for (int t = 0; t < places; t++) {
            wait_lds_loads<(AHEAD - 1) * NL>();
            __builtin_amdgcn_wave_barrier();
            const int cell0 = cell_of(t), b = (t >> 2) % GB;
            f4 part[TYPE == kF32 ? 4 : 1];
#pragma unroll
            for (int e = 0; e < (TYPE == kF32 ? 4 : 1); e++) part[e] = f4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < C::NK; j++) {
                const u4 kf = *reinterpret_cast<const u4 *>(&ring[wave][buf][m * ROWB + (((4 * j + g) ^ (m & SWAP)) << 4)]);
                if constexpr (TYPE == kF32) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[e]), __uint_as_float(qf[j][e]), part[e], 0, 0, 0);
                } else {
                    part[0] = mfma16<TYPE>(kf, qf[j], part[0]);
                }
            }
            f4 sc = part[0];
            if constexpr (TYPE == kF32) sc = (part[0] + part[1]) + (part[2] + part[3]);
            const f4 bias = *reinterpret_cast<const f4 *>(&cell_bias[wave][b][16 * (t & 3) + 4 * g]);
            float p[4];
            // (the difference before log2 e: its rounding goes with the weight's size, not the score's)
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = exp_of(__builtin_fmaf(sc[i], a.scale, bias[i]) - lse);
            if (cell0 + 16 > clear || (cell0 + 16 > a.first && cell0 < cut) || nothing) {
                const unsigned see = lse == -INFINITY ? 0 : seen32(a, q, tok, cell0) & window32(a, from, cell0);
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] = see >> (4 * g + i) & 1 ? p[i] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = bias[i] == -INFINITY ? 0.0f : p[i];
            // over the rows: lane m of the 16 gets cell m % 4's
            auto dpp = [](float x, auto ctrl) {
                return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true));
            };
            const float p0 = (m & 2 ? p[2] : p[0]) + dpp(m & 2 ? p[0] : p[2], std::integral_constant<int, 0x4e>{});
            const float p1 = (m & 2 ? p[3] : p[1]) + dpp(m & 2 ? p[1] : p[3], std::integral_constant<int, 0x4e>{});
            float x = (m & 1 ? p1 : p0) + dpp(m & 1 ? p0 : p1, std::integral_constant<int, 0xb1>{});
            x += dpp(x, std::integral_constant<int, 0x124>{});   // (rotations by four and eight lanes)
            x += dpp(x, std::integral_constant<int, 0x128>{});
            mine = m >> 2 == (t & 3) ? x : mine;
            if ((t & 3) == 3) {
                const int cell = cell0 - 48 + out_at;
                const float old = cell_old[wave][b][out_at];
                if (cell < q.held) w.weight[c.seq * w.w_seq + h * w.room + cell] = (row_lo ? old : w.decay * old) + mine;
            }
            // (what was read of this place is in registers: it may be filled again)
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
            fill();
            buf = buf + 1 < BUFS ? buf + 1 : 0;
        }
        wait_lds_loads<0>();
    }
}

template <int TYPE> bool run_weigh_ring(const WeighArgs & w, long long blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block(256);
    if (w.a.dk <= 64) return launch(k_weigh_ring<TYPE, 64>, grid, block, st, w);
    if (w.a.dk <= 128) return launch(k_weigh_ring<TYPE, 128>, grid, block, st, w);
    return launch(k_weigh_ring<TYPE, 256>, grid, block, st, w);
}

// More rows of 16-bit types: each of a block's four waves keeps the keys of 32
// cells in registers and goes over all rows, tiles of 64 in LDS. Rows reach LDS
// by direct loads, two tiles ahead (256-wide heads: one), pieces of 16 bytes exchanged by the row's
// number so that the lanes of a read are on different banks; the fragments are
// those of k_attn_tiles: a lane holds a row's scores of 16 of 32 cells. A tile is
// whole tokens: its rows' places are the same in every tile, and rows that are
// left over (or past the last token) repeat its last row with a log-sum-exp of
// +inf. RW = 2, for few blocks: eight waves, two a cell tile, over tiles of 128
// rows; they join in LDS.
//
// Without a bias the scores go into the exponential by one multiply-add (scale
// and log2 e in one factor). What that factor's rounding does to a score is done to
// the log-sum-exp too, by its own factor in two parts, so that it goes with their
// difference, and one rounding, of the log-sum-exp's product, with the score's size,
// as the score's own does in the other kernels. (With log2 e for the log-sum-exps:
// twice the error, scores of 5600 off by 3.4e-4 where half a step is 2.4e-4.)
//
// Bound by the exponentials: 512 of a tile's 900 cycles of vector instructions in
// a wave, its products 512 beside them. A prompt of 16384 tokens of 32 heads of
// 128: 1.19 to 1.30 ms by the card, 847 to 922 TFLOP/s (a large product: 1170 to
// 1240; with two waves a SIMD, 64 cells each, 1.40 ms); 32768 tokens 956 TFLOP/s,
// 4096 tokens, eight waves a block, 151 to 162 us (224 with four).
template <int TYPE, int D, bool BIAS, int RW>
__global__ __launch_bounds__(256 * RW, D == 256 || BIAS || RW == 2 ? 2 : 3) void k_weigh_tiles(WeighArgs w) {
    constexpr int CELLS = 128, ROWS = 64 * RW, KS = D / 16, CH = D / 8, ROWB = 2 * D;
    constexpr int SWAP = CH < 16 ? 7 : 15;                    // bits of a row's number that its pieces are exchanged by
    constexpr int WAVES = 4 * RW, NL = ROWS * CH / (64 * WAVES), RPL = 512 / D;   // direct loads of a wave and tile; rows of one
    constexpr int BUFS = D == 256 ? 2 : 3, AHEAD = BUFS - 1, LOADS = NL + 1;
    static_assert(BUFS * ROWS * ROWB <= 128 * 1024, "a block fits a CU");
    __shared__ __align__(16) char lds[BUFS][ROWS * ROWB];
    __shared__ float row_lse[BUFS][ROWS];
    __shared__ float join[RW == 2 ? 4 : 1][16][2];
    __shared__ int sums_nan[WAVES];

    const AttnArgs & a = w.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cw = wave & 3, rw = wave >> 2, n = lane & 31, hf = lane >> 5;
    int u = blockIdx.x;
    const int h = u % a.H;
    u /= a.H;
    const int first_tile = u % w.cell_tiles, s = u / w.cell_tiles;
    Counted c;
    if (!counted_of(w, s, c)) return;
    const Sequence & q = c.q;
    const int page_mask = (1 << a.shift) - 1;
    const int T = ROWS / a.G;                                 // tokens of a tile
    const float to_log2 = w.to_log2;
    // places of a tile's rows: this lane's two, and those it loads
    int my_tok[2];
    bool my_on[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int row = 64 * rw + 32 * r + n;
        my_on[r] = row < T * a.G;
        my_tok[r] = (my_on[r] ? row : T * a.G - 1) / a.G;
    }
    int load_tok[NL];
    unsigned load_off[NL];
    bool load_on[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int at = (i * WAVES + wave) * RPL + lane / CH, row = at < T * a.G ? at : T * a.G - 1;
        const int piece = (lane % CH) ^ (at & SWAP);
        load_tok[i] = row / a.G;
        load_off[i] = (unsigned)(row % a.G) * (unsigned)(2 * a.q_head) + 16 * piece;
        load_on[i] = 8 * piece < a.dk;
    }
    const int lse_at = 16 * wave + (lane & 15), lse_row = lse_at < T * a.G ? lse_at : T * a.G - 1;   // (lanes 0 .. 15)
    const int lse_tok = lse_row / a.G;
    const unsigned lse_off = 4 * (unsigned)(lse_row % a.G), lse_step = 4 * (unsigned)(a.H * a.G);

    for (int tile = first_tile; (long long)tile * CELLS < q.held; tile += w.cell_tiles) {
        const int block0 = tile * CELLS, cell0 = block0 + 32 * cw;
        int t0, t1;   // the block's tokens, and the wave's
        tokens_of(a, c, block0, block0 + CELLS < q.held ? block0 + CELLS : q.held, t0, t1);
        int wt0, wt1;
        tokens_of(a, c, cell0, cell0 + 32 < q.held ? cell0 + 32 : q.held, wt0, wt1);
        if (cell0 >= q.held) wt1 = wt0;

        // the next tile to load: its first token, its place, its rows and log-sum-exps
        int load_tt, load_buf;
        const char *load_q, *load_l;
        const long long q_step = 2 * T * a.q_tok, l_step = 4LL * T * a.H * a.G;
        auto fill = [&] {
            const int most = t1 - 1 - load_tt;
            char * to = lds[load_buf];
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int tk = load_tok[i] < most ? load_tok[i] : most;
                if (load_on[i]) load_lds16(load_q, load_off[i] + __umul24(tk, (unsigned)(2 * a.q_tok)), to + (i * WAVES + wave) * 1024);
            }
            if (lane < 16)
                load_lds4(load_l, lse_off + __umul24(lse_tok < most ? lse_tok : most, lse_step), reinterpret_cast<char *>(&row_lse[load_buf][16 * wave]));
            load_buf = load_buf + 1 < BUFS ? load_buf + 1 : 0;
            if (load_tt + T < t1) {   // (past the last tile: the last again, for the count of loads)
                load_tt += T;
                load_q += q_step;
                load_l += l_step;
            }
        };

        __syncthreads();   // (LDS of the last tile of cells is read)
        if (a.dk < D) {
            for (int i = threadIdx.x; i < BUFS * ROWS * CH; i += 64 * WAVES) reinterpret_cast<u4 *>(lds)[i] = u4{0, 0, 0, 0};
            __syncthreads();
        }
        u4 kf[KS];
        f16x bias, sum;
        unsigned there;   // cells of this lane's registers that rows may see
        {
            const int cell = cell0 + (n & 16);
            int page = cell < q.held ? q.table[cell >> a.shift] : -1;
            const bool good = page >= 0 && page < a.n_pages;
            if (!good) page = 0;
            const unsigned long long row = ((unsigned)page << a.shift) + ((cell + (n & 15)) & page_mask);
            const char * p = a.k.base + h * a.k.ld_head + row * a.k.ld_tok + 16 * hf;
            if (a.dk == D) {
#pragma unroll
                for (int j = 0; j < KS; j++) kf[j] = *reinterpret_cast<const u4 *>(p + 32 * j);
            } else {
#pragma unroll
                for (int j = 0; j < KS; j++)
                    kf[j] = 16 * j + 8 * hf < a.dk ? *reinterpret_cast<const u4 *>(p + 32 * j) : u4{0, 0, 0, 0};
            }
            const int left = q.held - cell0;
            const unsigned long long ok = __ballot(good);   // (lanes 0 and 16: the two groups of 16 cells)
            there = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
            there &= (ok & 1 ? 0xffffu : 0u) | (ok >> 16 & 1 ? 0xffff0000u : 0u);
            if constexpr (BIAS) {
                const int pages[2] = {__shfl(page, 0), __shfl(page, 16)};
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const int at = cell0 + 8 * y + 4 * hf;
                    const f4 b = *reinterpret_cast<const f4 *>(a.bias + (((long long)pages[y >> 1] * a.H + h) << a.shift) + (at & page_mask));
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        bias[4 * y + i] = b[i];
                        if (b[i] == -INFINITY) there &= ~(1u << (8 * y + 4 * hf + i));
                    }
                }
            }
        }
        auto arrive = [&] {
            wait_lds_loads<(AHEAD - 1) * LOADS>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            fill();
        };
        auto step = [&](int tt, int buf, auto kind) {
            constexpr bool PLAIN = decltype(kind)::value;
            f16x sc[2];
            float l2[2];   // (with a bias the log-sum-exp itself)
            unsigned see[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
#pragma unroll
                for (int i = 0; i < 16; i++) sc[r][i] = 0.0f;
                const float lse = row_lse[buf][64 * rw + 32 * r + n];
                const float less = BIAS ? lse : __builtin_fmaf(lse, w.lse_log2[0], lse * w.lse_log2[1]);
                l2[r] = fabsf(lse) == INFINITY || !my_on[r] || tt + my_tok[r] >= t1 ? INFINITY : less;
                if constexpr (!PLAIN) {
                    const int tok = tt + my_tok[r] < t1 ? tt + my_tok[r] : t1 - 1;
                    see[r] = lse == -INFINITY ? 0 : (seen32(a, q, tok, cell0) & window32(a, window_from(a, q, tok), cell0)) >> (4 * hf);
                }
            }
            // four of a row's scores to weights (PLAIN: exponentials side by side, with products around them)
            auto weights = [&](int r, int y) {
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    // (with a bias the difference first: a score may be the type's lowest value)
                    p[i] = BIAS ? exp_of(__builtin_fmaf(sc[r][4 * y + i], a.scale, bias[4 * y + i]) - l2[r])
                                : __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][4 * y + i], to_log2, -l2[r]));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (!PLAIN) p[i] = see[r] >> (8 * y + i) & 1 ? p[i] : 0.0f;
                    sum[4 * y + i] += p[i];
                }
            };
            auto row_part = [&](int r, int j) {
                return *reinterpret_cast<const u4 *>(&lds[buf][(64 * rw + 32 * r + n) * ROWB + (((2 * j + hf) ^ (n & SWAP)) << 4)]);
            };
            constexpr int PART = KS < 8 ? KS : 8;   // reads of LDS ahead of their products
            u4 qf[PART];
#pragma unroll
            for (int j0 = 0; j0 < KS; j0 += PART) {
#pragma unroll
                for (int j = 0; j < PART; j++) qf[j] = row_part(0, j0 + j);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < PART; j++) sc[0] = mfma32<TYPE>(kf[j0 + j], qf[j], sc[0]);
            }
#pragma unroll
            for (int j = 0; j < PART; j++) qf[j] = row_part(1, j);
            __builtin_amdgcn_sched_barrier(0);
            // the second rows' products run under the first ones' exponentials
#pragma unroll
            for (int y = 0; y < 4; y++) {
#pragma unroll
                for (int j = y * PART / 4; j < (y + 1) * PART / 4; j++) sc[1] = mfma32<TYPE>(kf[j], qf[j], sc[1]);
                weights(0, y);
                if constexpr (PLAIN) __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j0 = PART; j0 < KS; j0 += PART) {
#pragma unroll
                for (int j = 0; j < PART; j++) qf[j] = row_part(1, j0 + j);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < PART; j++) sc[1] = mfma32<TYPE>(kf[j0 + j], qf[j], sc[1]);
            }
#pragma unroll
            for (int y = 0; y < 4; y++) {
                weights(1, y);
                if constexpr (PLAIN) __builtin_amdgcn_sched_barrier(0);
            }
        };
        // Tiles whose rows all see all of this wave's cells begin at tokens w_lo .. w_hi - 1. (A
        // last tile of fewer tokens may be taken for one that does not.)
        int w_lo, w_hi;
        if (a.mask) {
            const int from = q.base - (q.n_new < a.last ? a.last - q.n_new : 0);
            w_lo = t0;
            w_hi = cell0 + 32 <= q.base && !(cell0 + 32 > a.first && cell0 < from) ? t1 : t0;
        } else {
            w_lo = cell0 + 31 - q.base;
            w_hi = cell0 + 32 > a.first && cell0 - q.base + a.last - T + 1 < t1 ? cell0 - q.base + a.last - T + 1 : t1;
        }
        if (w_hi <= w_lo) w_lo = w_hi = t1;
        int tt, buf;
        auto next = [&] {
            tt += T;
            buf = buf + 1 < BUFS ? buf + 1 : 0;
        };
        for (bool again = false;; again = true) {
            const int tok_lo = opaque(t0);
            load_tt = tok_lo;
            load_buf = 0;
            load_q = a.q + 2 * ((long long)(q.tok0 + tok_lo) * a.q_tok + (long long)(h * a.G) * a.q_head);
            load_l = reinterpret_cast<const char *>(a.lse + (long long)(q.tok0 + tok_lo) * a.H * a.G + h * a.G);
#pragma unroll
            for (int i = 0; i < 16; i++) sum[i] = 0.0f;
            if (t0 < t1) {
#pragma unroll
                for (int i = 0; i < AHEAD; i++) fill();
            }
            // (the keys are waited for here: a wait in the loop would be one for the rows on their way too)
#pragma unroll
            for (int j = 0; j < KS; j++) asm volatile("" : "+v"(kf[j]));
            tt = tok_lo;
            buf = 0;
            while (tt < t1) {
                const int stop = tt >= w_hi ? t1 : w_lo < t1 ? w_lo : t1;
                while (tt < stop) {
                    arrive();
                    if (tt + T > wt0 && tt < wt1) step(tt, buf, std::false_type{});
                    next();
                }
                while (tt < w_hi && tt < t1) {
                    arrive();
                    step(tt, buf, std::true_type{});
                    next();
                }
            }
            wait_lds_loads<0>();
            if (again) break;
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = there >> (8 * (i >> 2) + 4 * hf + (i & 3)) & 1 ? sum[i] : 0.0f;
            if (!any_nan(v, sums_nan)) break;
            w_lo = w_hi = t1;
        }
        // over a half's 32 lanes: each step hands half of the sums to the lane across, until each holds one cell's
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = there >> (8 * (i >> 2) + 4 * hf + (i & 3)) & 1 ? sum[i] : 0.0f;
#pragma unroll
        for (int m = 8; m; m >>= 1)
#pragma unroll
            for (int i = 0; i < m; i++) {
                const float mine = n & m ? v[m + i] : v[i], theirs = n & m ? v[i] : v[m + i];
                v[i] = mine + __shfl_xor(theirs, m);
            }
        v[0] += __shfl_xor(v[0], 16);
        if constexpr (RW == 2) {
            if (rw == 1 && n < 16) join[cw][n][hf] = v[0];
            __syncthreads();
            if (rw == 0 && n < 16) v[0] += join[cw][n][hf];
        }
        if (rw == 0 && n < 16) add_weight(w, c, h, cell0 + 8 * (n >> 2) + 4 * hf + (n & 3), v[0]);
    }
}

template <int TYPE, int D, int RW> bool run_weigh_tiles(const WeighArgs & w, long long blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block(256 * RW);
    return w.a.bias ? launch(k_weigh_tiles<TYPE, D, true, RW>, grid, block, st, w)
                    : launch(k_weigh_tiles<TYPE, D, false, RW>, grid, block, st, w);
}
template <int TYPE, int RW> bool run_weigh_tiles(const WeighArgs & w, long long blocks, hipStream_t st) {
    if (w.a.dk <= 64) return run_weigh_tiles<TYPE, 64, RW>(w, blocks, st);
    if (w.a.dk <= 128) return run_weigh_tiles<TYPE, 128, RW>(w, blocks, st);
    return run_weigh_tiles<TYPE, 256, RW>(w, blocks, st);
}
template <int TYPE> bool run_weigh_tiles(const WeighArgs & w, long long blocks, hipStream_t st) {
    return blocks <= 512 ? run_weigh_tiles<TYPE, 2>(w, blocks, st) : run_weigh_tiles<TYPE, 1>(w, blocks, st);
}

template <int TYPE, int QT, int D, bool SPLIT> bool run_weigh(const WeighArgs & w, bool careful, long long blocks, hipStream_t st) {
    constexpr int RT = TYPE == kF32 ? kFewRows32 : kFewRows16;
    const dim3 grid((unsigned)blocks), block(256);
    if constexpr (TYPE != kQ8)
        if (careful) return launch(k_weigh_rows<TYPE, QT, D, RT, ANY, SPLIT>, grid, block, st, w);
    if (w.a.dk == D) return launch(k_weigh_rows<TYPE, QT, D, RT, FULL, SPLIT>, grid, block, st, w);
    return launch(k_weigh_rows<TYPE, QT, D, RT, PART, SPLIT>, grid, block, st, w);
}
template <int TYPE, int QT, bool SPLIT> bool run_weigh(const WeighArgs & w, bool careful, long long blocks, hipStream_t st) {
    if (w.a.dk <= 64) return run_weigh<TYPE, QT, 64, SPLIT>(w, careful, blocks, st);
    if (w.a.dk <= 128) return run_weigh<TYPE, QT, 128, SPLIT>(w, careful, blocks, st);
    return run_weigh<TYPE, QT, 256, SPLIT>(w, careful, blocks, st);
}
template <int TYPE, int QT> bool run_weigh(const WeighArgs & w, bool split, bool careful, long long blocks, hipStream_t st) {
    return split ? run_weigh<TYPE, QT, true>(w, careful, blocks, st) : run_weigh<TYPE, QT, false>(w, careful, blocks, st);
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
    w.weight = y->weight + (long long)x->layer * c->max_seqs * w.w_seq;
    w.decay = y->decay;
    w.tail = y->tail;
    w.fresh = y->fresh;
    w.to_log2 = a.scale * kLog2e;
    {
        // (scales that leave no whole fraction of a float: scores are 0 then, or not finite)
        const double near = (double)w.to_log2 / a.scale, of = near > 1.4 && near < 1.5 ? near : 1.44269504088896340736;
        w.lse_log2[0] = (float)of;
        w.lse_log2[1] = (float)(of - w.lse_log2[0]);
    }
    const int es = esize(x->type);
    const bool careful = c->k_type != kQ8 && (!vec_rows(x->q, es) || c->d_k * es % 16);
    const long long rows = (long long)(y->tail > 0 && y->tail < x->max_new ? y->tail : x->max_new) * a.G;
    const bool few = rows <= 16 * (c->k_type == kF32 ? kFewRows32 : kFewRows16);
    const bool ring = rows <= 16 && !careful && c->k_type != kQ8;
    // (strides that direct loads take)
    const bool tiles = !few && a.G <= 64 && !careful && (c->k_type == kF16 || c->k_type == kBF16) && x->q.ld_tok >= 0 &&
                       x->q.ld_tok < 1 << 23 && x->q.ld_head >= 0 && x->q.ld_head < 1 << 23 && x->n_head < 1 << 20;
    const long long units = (long long)x->n_seq * c->n_head_kv;
    const long long most = kMaxBlocks / units;
    if (most < 1) return KV_COMPACT_E_UNSUPPORTED;
    // Blocks: 128 cells each where rows come by tiles or 16 at a time. Otherwise
    // ranges of at least 512 cells (up to 16 rows; 256 above), or half of that
    // where it leaves fewer than 512 blocks, and not more than fill the GPU many
    // times. Measured, us (8 x 128, bf16; one token, ranges of 128, 256 and 512):
    // one sequence of 2000 cells 6.5, 6.6 and 8.7, of 20000 15.9, 12.7 and 12.6;
    // 16 of 2000 18.8, 13.8 and 11.4; 64 of up to 16384, 4096, 8192 and 16384
    // blocks: 278, 266 and 262. 32 tokens, ranges of 128 and 256: one of 20000
    // 24.5 and 21.6, 4 of 4096 15.4 and 17.4. Above 16 rows, or over Q8_0, ten
    // blocks a CU, an odd number of ranges of each sequence (an even one keeps a
    // CU at the same range of every sequence): 2048, 2560 and 4096 blocks, 32
    // tokens, 8 of up to 20000 55, 53 and 60, 24 of up to 16000 134, 133 and 132;
    // Q8_0, one token, 64 of up to 16384 in 4, 5, 7 and 8 ranges 312, 246, 230 and
    // 256, 128 of up to 8192 in 2, 3 and 4 ranges 309, 231 and 307: the rule takes 5,
    // where 7 would be faster, and 3. Under a window all cells' keys are read here all
    // the same, and hidden ones multiplied for nothing.
    long long want = ((long long)x->max_len + 127) / 128;
    if (few) {
        const int least = ring ? 512 : 256, fill = ring ? 16384 : 2560;
        want = ((long long)x->max_len + least - 1) / least;
        if (want * units < 512) want = ((long long)x->max_len + least / 2 - 1) / (least / 2);
        const long long enough = (fill + units - 1) / units;
        want = want < enough ? want : ring ? enough : enough | 1;
    }
    const bool split = !few && !tiles && want * units < kSplit;
    if (split) want = ((long long)x->max_len + 31) / 32;
    w.cell_tiles = (int)(want < 1 ? 1 : want < most ? want : most);
    const int group = ring ? 64 : 32;
    w.range = (int)(((long long)x->max_len + (long long)group * w.cell_tiles - 1) / ((long long)group * w.cell_tiles));
    w.a = a;
    const long long blocks = units * w.cell_tiles;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    bool ok;
    if (ring) {
        ok = c->k_type == kF32 ? run_weigh_ring<kF32>(w, blocks, st)
             : c->k_type == kF16 ? run_weigh_ring<kF16>(w, blocks, st)
                                 : run_weigh_ring<kBF16>(w, blocks, st);
    } else if (few) {
        if (c->k_type == kF32) ok = run_weigh_few<kF32, kF32>(w, rows, careful, blocks, st);
        else if (c->k_type == kF16) ok = run_weigh_few<kF16, kF16>(w, rows, careful, blocks, st);
        else if (c->k_type == kBF16) ok = run_weigh_few<kBF16, kBF16>(w, rows, careful, blocks, st);
        else if (x->type == kF16) ok = run_weigh_few<kQ8, kF16>(w, rows, careful, blocks, st);
        else ok = run_weigh_few<kQ8, kBF16>(w, rows, careful, blocks, st);
    } else if (tiles) {
        ok = c->k_type == kF16 ? run_weigh_tiles<kF16>(w, blocks, st) : run_weigh_tiles<kBF16>(w, blocks, st);
    } else if (c->k_type == kF32) ok = run_weigh<kF32, kF32>(w, split, careful, blocks, st);
    else if (c->k_type == kF16) ok = run_weigh<kF16, kF16>(w, split, careful, blocks, st);
    else if (c->k_type == kBF16) ok = run_weigh<kBF16, kBF16>(w, split, careful, blocks, st);
    else if (x->type == kF16) ok = run_weigh<kQ8, kF16>(w, split, careful, blocks, st);
    else ok = run_weigh<kQ8, kBF16>(w, split, careful, blocks, st);
    return ok ? 0 : KV_COMPACT_E_DEVICE;
}
