// Attention kernels on MI355X (include/kvc-cache.h): new or drafted tokens
// over a paged cache, and whole prompts.
//
// One pass over the keys with a running maximum and sum per row:
//   s = scale q.k + bias, m' = max(m, max s), a = exp(m - m'),
//   p = exp(s - m'), l' = a l + sum p, o' = a o + p V; result o / l, lse m + log l.
// The products run on matrix instructions in the transposed form
//   S^T[key][row] = K Q^T,  O^T[column][row] = V^T P^T,
// because a lane then holds one row in both: the scores it gets from the first
// product are, as they lie in its registers, its part of the second one's
// operand, and the row's maximum, sum and rescale need no transposition.
//
// Rows of a KV head are its tokens times the group's query heads, so that a
// key is read once for all of them.
#include "kvc_launch.h"

#include <math.h>
#include <stdint.h>

#include <type_traits>

// (the library is built with contraction off for the kernels that keep the
// reference's rounding; a multiply-add here may be one rounding)
#pragma clang fp contract(fast)

namespace kvc {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kF32 = KV_TYPE_F32, kF16 = KV_TYPE_F16, kBF16 = KV_TYPE_BF16, kQ8 = KV_TYPE_Q8_0;

// Where rows of K or V stand: pages of a pool (table set), or one array.
struct RowsAt {
    const char * base;
    long long ld_head;   // bytes
    unsigned ld_tok;     // bytes, under 2^24
};

struct AttnArgs {
    RowsAt k, v;
    const char * q;
    char * o;
    long long q_tok, q_head, o_tok, o_head;   // elements
    float * lse;
    const int * cu;
    const int * seqs;
    const int * len;       // cells of each sequence, or nullptr: its tokens
    const int * table;     // pages, or nullptr: contiguous tokens
    const float * bias;    // this layer's [page][H][page_size], or nullptr
    const unsigned long long * mask;
    int mask_words, n_seq, n_tok, H, G, dk, dv;
    int shift, n_pages, max_seqs, max_pages;
    int splits, range;     // key ranges of at least `range` keys: a short sequence fills the first few
    int tiles;             // row tiles the grid has for each sequence (0: flat over all sequences)
    float scale;
    float * part_o;        // [splits][n_tok * n_head][dv]
    float * part_ml;       // [splits][n_tok * n_head][2]
};

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// Exchange between lane groups 16 and 32 apart: the larger (sum) of the four
// lanes that hold one row.
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float row_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

__device__ __forceinline__ float f16_value(unsigned short u) { return (float)__builtin_bit_cast(_Float16, u); }
__device__ __forceinline__ float bf16_value(unsigned short u) { return __uint_as_float((unsigned)u << 16); }

template <int TYPE> __device__ __forceinline__ float value_of(const char * p, long long i) {
    if constexpr (TYPE == kF32) return reinterpret_cast<const float *>(p)[i];
    const unsigned short u = reinterpret_cast<const unsigned short *>(p)[i];
    if constexpr (TYPE == kBF16) return bf16_value(u);
    return f16_value(u);
}

// two fp32 values rounded (to nearest even) into one register of the 16-bit type
template <int TYPE> __device__ __forceinline__ unsigned pack2(float a, float b) {
    if constexpr (TYPE == kF16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        h2 r = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(unsigned, r);
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        b2 r = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(unsigned, r);
    }
}

template <int TYPE> __device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c) {
    if constexpr (TYPE == kF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// loads from 2-byte boundaries (one instruction each: the memory takes any address)
typedef u4 u4_any __attribute__((aligned(2)));
typedef u2 u2_any __attribute__((aligned(2)));
typedef unsigned u1_any __attribute__((aligned(2)));

// How the columns of a row are read: FULL the heads are as wide as the form,
// PART rows are 16-byte aligned and heads whole vectors, ANY element by element.
enum Columns { FULL, PART, ANY };

// N elements (16 bytes, or 8) from column `col` of a row of d that stands at
// base + row. Nothing is read at or past column d: zeros there.
template <int N, int BYTES, Columns COLS>
__device__ __forceinline__ void load_cols(const char * base, unsigned row, int col, int d, unsigned * out) {
    constexpr int W = N * BYTES / 4;
    if constexpr (COLS != ANY) {
        if (COLS == FULL || col < d) {
            if constexpr (W == 4)
                *reinterpret_cast<u4 *>(out) = *reinterpret_cast<const u4 *>(base + (row + (unsigned)col * BYTES));
            else
                *reinterpret_cast<u2 *>(out) = *reinterpret_cast<const u2 *>(base + (row + (unsigned)col * BYTES));
        } else {
            for (int i = 0; i < W; i++) out[i] = 0;
        }
    } else {
        for (int i = 0; i < W; i++) {
            if constexpr (BYTES == 4) {
                out[i] = col + i < d ? reinterpret_cast<const unsigned *>(base + row)[col + i] : 0;
            } else {
                const unsigned short * r = reinterpret_cast<const unsigned short *>(base + row);
                const unsigned a = col + 2 * i < d ? r[col + 2 * i] : 0, b = col + 2 * i + 1 < d ? r[col + 2 * i + 1] : 0;
                out[i] = a | b << 16;
            }
        }
    }
}

// a table entry at a uniform address, by a scalar load (nothing writes tables while attention runs)
__device__ __forceinline__ int uniform_load(const int * p) {
    return *(const __attribute__((address_space(4))) int *)p;
}

// A sequence of the call: its tokens, and the keys it holds.
struct Sequence {
    int tok0, n_new;
    int held;            // keys; 0: nothing can be seen
    int base;            // keys that every token sees
    const int * table;   // pages, or nullptr: contiguous tokens
};
__device__ __forceinline__ Sequence sequence_of(const AttnArgs & a, int s) {
    Sequence q;
    int tok0 = uniform_load(a.cu + s), tok1 = uniform_load(a.cu + s + 1);
    tok0 = tok0 < 0 ? 0 : tok0;
    tok1 = tok1 > a.n_tok ? a.n_tok : tok1;
    q.tok0 = tok0;
    q.n_new = tok1 - tok0;
    q.held = q.n_new;
    q.table = nullptr;
    if (a.table) {
        const int seq = a.seqs ? uniform_load(a.seqs + s) : s;
        const bool there = seq >= 0 && seq < a.max_seqs;
        q.held = there ? uniform_load(a.len + seq) : 0;
        if (q.held < q.n_new || q.held > (long long)a.max_pages << a.shift) q.held = 0;
        q.table = a.table + (long long)(there ? seq : 0) * a.max_pages;
    }
    q.base = q.held ? q.held - q.n_new : 0;
    return q;
}

// Tiles of a key range, of n_tiles in all. Ranges of the same size for all
// sequences are blocks of the same length; more keys than the launch was told
// of make them longer.
__device__ __forceinline__ int range_tiles(const AttnArgs & a, int n_tiles, int keys) {
    const int even = (n_tiles + a.splits - 1) / a.splits, said = (a.range + keys - 1) / keys;
    return even > said ? even : said;
}

// The u-th tile of `rows` rows of all sequences together, those of a sequence
// from its end (the most keys first). False past the last one.
__device__ __forceinline__ bool find_tile(const AttnArgs & a, int u, int rows, int lane, int & s, int & tile) {
    int before = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
        int tiles = 0;
        if (s0 + lane < a.n_seq) {
            const int n = a.cu[s0 + lane + 1] - a.cu[s0 + lane];
            tiles = n > 0 ? (int)(((long long)n * a.G + rows - 1) / rows) : 0;
        }
        int incl = tiles;
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(incl, o);
            if (lane >= o) incl += y;
        }
        const unsigned long long hit = __ballot(before + incl > u);
        if (hit) {
            const int w = __ffsll((long long)hit) - 1;
            s = s0 + w;
            tile = __shfl(tiles, w) - 1 - (u - before - (__shfl(incl, w) - __shfl(tiles, w)));
            return true;
        }
        before += __shfl(incl, 63);
    }
    return false;
}

// Bit i: token `tok` of a sequence sees key key0 + i (its score's bias and its page apart)
__device__ __forceinline__ unsigned seen32(const AttnArgs & a, const Sequence & q, int tok, int key0) {
    auto first = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; };
    const unsigned all = first(q.held - key0);
    const int rel = key0 - q.base;
    if (rel <= -32) return all;
    if (!a.mask) return all & first(tok - rel + 1);
    const unsigned long long * w = a.mask + (long long)(q.tok0 + tok) * a.mask_words;
    auto word = [&](int i) { return i < a.mask_words ? w[i] : 0ull; };
    if (rel < 0) return all & ((unsigned)(word(0) << -rel) | first(-rel));
    const int i = rel >> 6, sh = rel & 63;
    unsigned long long bits = word(i) >> sh;
    if (sh > 32) bits |= word(i + 1) << (64 - sh);
    return all & (unsigned)bits;
}

// 16 bytes a lane from memory to LDS, lane l's to `to` + 16 l (`from` and `to`
// uniform; lanes that are off leave theirs as it is). The compiler does not
// count these loads: wait_lds_loads() does.
__device__ __forceinline__ void load_lds16(const char * from, unsigned offset, char * to) {
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)to;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(from), "s"(at) : "m0", "memory");
}
// (4 bytes, each from an address of its own)
__device__ __forceinline__ void load_lds4(const char * from, char * to) {
    const unsigned at = __builtin_amdgcn_readfirstlane(
        (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)to);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(at) : "m0", "memory");
}
// until at most N of the wave's loads are on their way
template <int N> __device__ __forceinline__ void wait_lds_loads() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
// Two signed bytes, chosen by `pick` (as v_perm: 0-3 of b, 4-7 of a; the other
// halves' bytes 0x0c), as exact fp16: byte + 128 is the low byte of 1024 + it.
__device__ __forceinline__ unsigned code_pair(unsigned a, unsigned b, unsigned pick) {
    const unsigned w = __builtin_amdgcn_perm(a, b, pick) ^ 0x64806480u;
    const h2 x = __builtin_bit_cast(h2, w) - h2{(_Float16)1152.0f, (_Float16)1152.0f};
    return __builtin_bit_cast(unsigned, x);
}

// signed byte i of a register pair, as fp32
__device__ __forceinline__ float byte_value(const unsigned * w, int i) {
    return (float)(int)(signed char)(w[i >> 2] >> (8 * (i & 3)));
}

// Attention of RT tiles of 16 rows (of one KV head of one sequence) over a
// range of keys; four waves of a block take alternate tiles of 32 keys and
// join in LDS. TYPE: the type of the cache rows (kQ8: q and o are QT).
// D: 64, 128 or 256, the head widths rounded up.
//
// Fragments (16x16x32, lane l, m = l % 16, g = l / 16): an operand's lane
// holds row m and elements 8g .. 8g+7 of the summed axis, a result's lane
// column m and rows 4g .. 4g+3. Keys of a 32-key tile are numbered on the
// summed axis of the second product so that a lane's elements are the scores
// it holds: 4g+i of the first 16 keys, then of the second. V's lane m holds
// VW neighbouring columns of those keys, which makes VW fragments after a
// 2 x 2 exchange of halves (v_perm), without LDS.
// F32 sums 4 elements an instruction (16x16x4), one of them a lane's.
// Q8_0: products in fp16, which holds the codes exactly. A block of K is one
// instruction, and its scale multiplies the block's sums in fp32; bf16 queries
// become fp16 times a power of two of their row. V is scale times code in fp16
// (for fp16 results with the remainder as a second term), which is a half step
// off at most while the scales are between 2^-14 and 2^8; a tile with others
// multiplies in fp32 (16x16x4).
//
// Each key is read once for all rows of its head, straight into the registers
// the products take it from, a tile ahead. One token of 64 sequences of up to
// 16384 bf16 cells (8 x 128, 32 heads): 0.52 ms, 5.2 TB/s (a plain read: 6.8).
// One sequence of 4096 cells: 14 us with the join, two launches and two
// latencies; of 20000 F32 cells with a bias: 49 us, 3.4 TB/s. Trees of 13 tokens
// of 32 heads over 16 sequences of up to 32768 Q8_0 cells (8 x 128): 409 us.
// Four row tiles a wave decode a key once for all 52 rows and leave one wave a
// SIMD: vector instructions are 47 % of its cycles, matrix instructions 9 %,
// and most of the rest is loads that nothing else runs under.
template <int TYPE, int QT, int D, int RT, Columns COLS>
struct RowKernel {
    static constexpr int ES = TYPE == kF32 ? 4 : 2;          // bytes of a q element
    static constexpr int KV = 16 / ES;                       // q / k elements a 16-byte load holds
    static constexpr int NK = D / (4 * KV);                  // loads of a q or k row
    static constexpr int VW = TYPE == kF32 ? 4 : (D / 16 < 8 ? D / 16 : 8);
    static constexpr int NU = D / 16 / VW;                   // V loads of a row
    static constexpr int NC = D / 16;                        // column fragments
    static constexpr int NB = D / 32;                        // Q8_0 blocks
    static constexpr bool Q8 = TYPE == kQ8;
    static constexpr int WV = Q8 ? (VW + 3) / 4 : VW * ES / 4;    // registers of a V load
    static constexpr int WK = Q8 ? 2 : 4;
    static constexpr int NKL = Q8 ? NB : NK;
    static constexpr int MT = Q8 ? kF16 : TYPE;              // type on the matrix units

    // fp16 weights are 2^10 times exp(s - m): those under 2^-24 of the largest, not 2^-14, lose bits
    static constexpr float lift = MT == kF16 ? 0x1p10f : 1.0f;
    static constexpr float log_lift = MT == kF16 ? 6.93147180559945309417f : 0.0f;

    // column of fragment c's lane m
    static __device__ __forceinline__ int column(int m, int c) { return (c / VW) * 16 * VW + VW * m + c % VW; }
};

// Tiles of a block's key range that left out values which are not finite: a bit
// for each of up to 64 stretches of 2^shift tiles.
struct OddTiles {
    int t_lo, t_hi, shift;
    unsigned long long bits = 0;
    __device__ __forceinline__ OddTiles(int lo, int hi) : t_lo(lo), t_hi(hi) {
        shift = hi - lo > 64 ? 26 - __builtin_clz(hi - lo - 1) : 0;
    }
    __device__ __forceinline__ void add(int t) { bits |= 1ull << ((t - t_lo) >> shift); }
    // f(first key, key past the last) of each stretch, tiles of `keys` keys
    template <class F> __device__ __forceinline__ void each(int keys, int held, F f) const {
#pragma nounroll
        for (unsigned long long m = bits; m; m &= m - 1) {
            const int t0 = t_lo + ((__ffsll((long long)m) - 1) << shift);
            const int t1 = t0 + (1 << shift) < t_hi ? t0 + (1 << shift) : t_hi;
            f(t0 * keys, t1 * keys < held ? t1 * keys : held);
        }
    }
};

// Values of V that are not finite, for the rows of tiles that left them out:
// one by one, the scores computed again.
template <int TYPE, int QT> struct Odd {
    const AttnArgs & a;
    const Sequence & q;
    int h, tok, head;

    __device__ __forceinline__ const char * row_of(const RowsAt & x, int key) const {
        long long row = q.tok0 + key;
        if (q.table) {
            const int p = q.table[key >> a.shift];
            if (p < 0 || p >= a.n_pages) return nullptr;
            row = ((long long)p << a.shift) + (key & ((1 << a.shift) - 1));
        }
        return x.base + h * x.ld_head + row * x.ld_tok;
    }
    static __device__ __forceinline__ float at(const char * row, int col) {
        if constexpr (TYPE == kQ8)
            return f16_value(*reinterpret_cast<const unsigned short *>(row + col / 32 * 34)) *
                   (float)*reinterpret_cast<const signed char *>(row + col / 32 * 34 + 2 + col % 32);
        else
            return value_of<TYPE>(row, col);
    }
    // weight (relative to exp(top)) times value where the value is not finite and the row sees its key, else 0
    __device__ __forceinline__ float term(int key, int col, float top) const {
        const char * v = row_of(a.v, key);
        if (!v) return 0.0f;
        const float x = at(v, col);
        if (fabsf(x) < INFINITY || !(seen32(a, q, tok, key) & 1)) return 0.0f;
        float b = 0.0f;
        if (a.bias)
            b = a.bias[(((long long)q.table[key >> a.shift] * a.H + h) << a.shift) + (key & ((1 << a.shift) - 1))];
        if (b == -INFINITY) return 0.0f;
        const char * k = row_of(a.k, key);
        const char * p = a.q + ((long long)(q.tok0 + tok) * a.q_tok + (long long)(h * a.G + head) * a.q_head) * (QT == kF32 ? 4 : 2);
        float s = 0.0f;
#pragma nounroll
        for (int i = 0; i < a.dk; i++) s += value_of<QT>(p, i) * at(k, i);
        return exp_of(s * a.scale + b - top) * x;
    }
};

template <int TYPE, int QT, int D, int RT, Columns COLS>
__global__ __launch_bounds__(256, D <= 128 && TYPE != kF32 && !(TYPE == kQ8 && D * RT > 128) ? 2 : 1) void k_attn_rows(AttnArgs a) {
    using C = RowKernel<TYPE, QT, D, RT, COLS>;
    constexpr int ROWS = 16 * RT, LD = D + 4;
    constexpr bool Q8 = C::Q8;
    __shared__ __align__(16) float join[4][ROWS][LD];
    __shared__ float join_m[4][ROWS], join_l[4][ROWS];
    __shared__ unsigned long long join_odd[4];
    // Q8_0 scales of a wave's tile, by block and key
    __shared__ __align__(16) float k_scale[Q8 ? 4 : 1][Q8 ? C::NB : 1][32];
    __shared__ __align__(16) _Float16 v_scale[Q8 ? 4 : 1][Q8 ? C::NB : 1][32];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4;

    // which rows: KV head h fastest, then the key range, the row tile, the sequence
    int u = blockIdx.x;
    const int h = u % a.H;
    u /= a.H;
    const int split = u % a.splits;
    u /= a.splits;
    int s = 0, tile = 0, tile_step;
    if (a.tiles) {
        tile = u % a.tiles;
        s = u / a.tiles;
        tile_step = a.tiles;
    } else {
        if (!find_tile(a, u, ROWS, lane, s, tile)) return;
        tile_step = 1 << 30;
    }
    s = __builtin_amdgcn_readfirstlane(s);
    tile = __builtin_amdgcn_readfirstlane(tile);
    const Sequence sq = sequence_of(a, s);
    if (sq.n_new <= 0) return;
    const int tok0 = sq.tok0, n_new = sq.n_new, held = sq.held, base = sq.base;
    const int * table = sq.table;
    const int rows = n_new * a.G;
    const int page_mask = a.table ? (1 << a.shift) - 1 : 0;

    for (; (long long)tile * ROWS < rows; tile += tile_step) {
        const int row0 = tile * ROWS;
        // keys this tile can see, and this block's range of them
        int last_tok = (row0 + ROWS - 1) / a.G;
        if (last_tok >= n_new) last_tok = n_new - 1;
        const int end_all = held == 0 ? 0 : (a.mask ? held : base + last_tok + 1);
        const int first_tok = row0 / a.G;
        const int clear = a.mask ? base : base + first_tok + 1;   // keys before it are seen by every row
        const int n_tiles = (end_all + 31) >> 5;
        const int per = range_tiles(a, n_tiles, 32);
        const int t_lo = split * per, t_hi = t_lo + per < n_tiles ? t_lo + per : n_tiles;

        // rows of this lane
        int tok[RT], head[RT];
        bool on[RT];
        u4 q[RT][C::NK];
        float to_score[RT], rest[RT];   // what turns a row's products into scores, in two parts (rest: 1 but for Q8_0 rows of extreme size)
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const int row = row0 + 16 * r + m;
            on[r] = row < rows;
            tok[r] = on[r] ? row / a.G : 0;
            head[r] = on[r] ? row % a.G : 0;
            to_score[r] = a.scale;
            rest[r] = 1.0f;
            const char * p = a.q + ((long long)(tok0 + tok[r]) * a.q_tok + (long long)(h * a.G + head[r]) * a.q_head) * C::ES;
#pragma unroll
            for (int j = 0; j < C::NK; j++) {
                const int col = 4 * C::KV * j + C::KV * g;
                if constexpr (Q8) {   // (the cache is aligned, the queries may not be)
                    q[r][j] = COLS == FULL || col < a.dk ? *reinterpret_cast<const u4_any *>(p + 2 * col) : u4{0, 0, 0, 0};
                } else {
                    unsigned w[4];
                    load_cols<C::KV, C::ES, COLS>(p, 0, col, a.dk, w);
                    q[r][j] = u4{w[0], w[1], w[2], w[3]};
                }
            }
            if constexpr (Q8 && QT == kBF16) {
                // the largest of the row to 2^14 (eight bits of it: exact; others from 2^-28 of it on)
                unsigned top = 0;
#pragma unroll
                for (int j = 0; j < C::NK; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const unsigned lo = q[r][j][i] & 0x7fffu, hi = q[r][j][i] >> 16 & 0x7fffu;
                        top = lo > top ? lo : top;
                        top = hi > top ? hi : top;
                    }
                top = max(top, (unsigned)__shfl_xor((int)top, 16));
                top = max(top, (unsigned)__shfl_xor((int)top, 32));
                int e = (int)(top >> 7) - 127;               // of the largest
                if (top == 0 || top >= 0x7f80u) e = 14;      // nothing, or not finite: as it is
                const int near = 14 - e > 100 ? 100 : 14 - e < -100 ? -100 : 14 - e;
                const float up = __builtin_ldexpf(1.0f, near), more = __builtin_ldexpf(1.0f, 14 - e - near);
#pragma unroll
                for (int j = 0; j < C::NK; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        q[r][j][i] = pack2<kF16>(bf16_value((unsigned short)q[r][j][i]) * up * more,
                                                 bf16_value((unsigned short)(q[r][j][i] >> 16)) * up * more);
                to_score[r] = a.scale * __builtin_ldexpf(1.0f, -near);
                rest[r] = __builtin_ldexpf(1.0f, near - (14 - e));
            }
        }
        f4 acc[RT][C::NC];
        float mx[RT], sum[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            mx[r] = -INFINITY;
            sum[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < C::NC; c++) acc[r][c] = f4{0, 0, 0, 0};
        }

        // pages of the two 16-cell groups of a tile (-1 past the end), and a group's first row
        auto pages_of = [&](int t, int (&pg)[2]) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int key = (t << 5) + 16 * x;
                pg[x] = !table ? 0 : t < t_hi && key < held ? uniform_load(table + (key >> a.shift)) : -1;
            }
        };
        auto good = [&](int pg) { return !table || (pg >= 0 && pg < a.n_pages); };
        // a group's first row (uniform), and the place of its row r behind it
        auto rows16 = [&](const RowsAt & x, int key, int pg) -> const char * {
            const unsigned row = table ? ((unsigned)(good(pg) ? pg : 0) << a.shift) + (key & page_mask)
                                       : (unsigned)(tok0 + (key < held ? key : held - 1));
            return x.base + h * x.ld_head + (unsigned long long)row * x.ld_tok;
        };
        auto row_of = [&](const RowsAt & x, int key, int r) -> unsigned {
            // (contiguous rows end with the sequence: those past it repeat the last)
            if (!table) r = key + r < held ? r : key < held ? held - 1 - key : 0;
            return (unsigned)__umul24(r, x.ld_tok);
        };

        unsigned kr[2][C::NKL][C::WK];
        unsigned vr[8][C::NU][C::WV];
        unsigned short ks[Q8 ? C::NB / 2 : 1], vsc[Q8 ? C::NB / 2 : 1];   // scales, a lane pair per key
        f4 bias[2];
        auto load_k = [&](int t, const int (&pg)[2]) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int key = (t << 5) + 16 * x;
                const char * p = rows16(a.k, key, pg[x]);
                const unsigned row = row_of(a.k, key, m);
#pragma unroll
                for (int j = 0; j < C::NKL; j++) {
                    if constexpr (Q8) {
                        *reinterpret_cast<u2 *>(kr[x][j]) =
                            COLS == FULL || 32 * j < a.dk ? *reinterpret_cast<const u2_any *>(p + (row + 34 * j + 2 + 8 * g)) : u2{0, 0};
                    } else {
                        load_cols<C::KV, C::ES, COLS>(p, row, 4 * C::KV * j + C::KV * g, a.dk, kr[x][j]);
                    }
                }
                // (four cells of one page)
                if (a.bias)
                    bias[x] = *reinterpret_cast<const f4 *>(
                        a.bias + (((long long)(good(pg[x]) ? pg[x] : 0) * a.H + h) << a.shift) + ((key + 4 * g) & page_mask));
            }
            if constexpr (Q8) {
                const int key = lane >> 1, half = lane & 1;
                const char * pk = key < 16 ? rows16(a.k, t << 5, pg[0]) : rows16(a.k, (t << 5) + 16, pg[1]);
                const char * pv = key < 16 ? rows16(a.v, t << 5, pg[0]) : rows16(a.v, (t << 5) + 16, pg[1]);
                pk += __umul24(key & 15, a.k.ld_tok) + 34 * half;
                pv += __umul24(key & 15, a.v.ld_tok) + 34 * half;
#pragma unroll
                for (int b = 0; b < C::NB / 2; b++) {
                    const int at = 2 * b + half;
                    ks[b] = COLS == FULL || 32 * at < a.dk ? *reinterpret_cast<const unsigned short *>(pk + 68 * b) : 0;
                    vsc[b] = COLS == FULL || 32 * at < a.dv ? *reinterpret_cast<const unsigned short *>(pv + 68 * b) : 0;
                }
            }
        };
        auto load_v = [&](int t, const int (&pg)[2]) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int key = (t << 5) + 16 * x;
                const char * p0 = rows16(a.v, key, pg[x]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const unsigned row = row_of(a.v, key, 4 * g + i);
#pragma unroll
                    for (int w = 0; w < C::NU; w++) {
                        const int col = C::column(m, w * C::VW);
                        if constexpr (Q8) {
                            const char * b = p0 + (row + col / 32 * 34 + 2 + col % 32);
                            if constexpr (C::WV == 2)
                                *reinterpret_cast<u2 *>(vr[4 * x + i][w]) = COLS == FULL || col < a.dv ? *reinterpret_cast<const u2_any *>(b) : u2{0, 0};
                            else
                                vr[4 * x + i][w][0] = COLS == FULL || col < a.dv ? *reinterpret_cast<const u1_any *>(b) : 0;
                        } else {
                            load_cols<C::VW, C::ES, COLS>(p0, row, col, a.dv, vr[4 * x + i][w]);
                        }
                    }
                }
            }
        };

        int page[2], next[2], later[2];
        f4 sc[RT][2];
        OddTiles odd_tiles(t_lo, t_hi);   // with values that are not finite (they are left out, and added at the end)
        // K of the next tile is loaded behind the first product, V behind the
        // second, page numbers a tile earlier: the loads run under the arithmetic
        pages_of(t_lo + wave, page);
        pages_of(t_lo + wave + 4, next);
        if (t_lo + wave < t_hi) {
            load_k(t_lo + wave, page);
            load_v(t_lo + wave, page);
        }
        // A tile that is not plain: a key hidden from some row, a bad page, Q8_0
        // scales that fp16 products do not hold, or not finite.
        auto special = [&](int t) {
            bool any = (t << 5) + 32 > clear || !good(page[0]) || !good(page[1]);
            bool mine = false;
            if (a.bias)
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int i = 0; i < 4; i++) mine |= bias[x][i] == -INFINITY;
            if constexpr (Q8)
#pragma unroll
                for (int b = 0; b < C::NB / 2; b++) {
                    const float v = fabsf(f16_value(vsc[b]));
                    mine |= v != 0.0f && !(v >= 0x1p-14f && v <= 256.0f);
                }
            return any || __ballot(mine) != 0;
        };
        auto step = [&](int t, auto kind) {
            constexpr bool SPECIAL = decltype(kind)::value;
            bool odd = false;
            const int key0 = t << 5;
            const bool ok[2] = {good(page[0]), good(page[1])};
            pages_of(t + 8, later);
            if constexpr (Q8) {
                // to the lanes that hold the blocks' sums and values; cells that are not there weigh nothing
                const int key = lane >> 1, half = lane & 1;
                const bool there = key0 + key < held && (key < 16 ? ok[0] : ok[1]);
#pragma unroll
                for (int b = 0; b < C::NB / 2; b++) {
                    k_scale[wave][2 * b + half][key] = f16_value(ks[b]);
                    unsigned short d = vsc[b];
                    if constexpr (SPECIAL) {
                        if (!there) d = 0;
                        if ((d & 0x7c00u) == 0x7c00u) {
                            odd = true;
                            d = 0;
                        }
                    }
                    v_scale[wave][2 * b + half][key] = __builtin_bit_cast(_Float16, d);
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }

            // S^T of both halves
#pragma unroll
            for (int x = 0; x < 2; x++) {
#pragma unroll
                for (int r = 0; r < RT; r++) sc[r][x] = f4{0, 0, 0, 0};
                if constexpr (TYPE == kF32) {
                    // (four sums of a quarter of the products each: shorter chains, and less rounding)
                    f4 part[RT][4];
#pragma unroll
                    for (int r = 0; r < RT; r++)
#pragma unroll
                        for (int e = 0; e < 4; e++) part[r][e] = f4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < C::NKL; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
#pragma unroll
                            for (int r = 0; r < RT; r++)
                                part[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __uint_as_float(kr[x][j][e]), __uint_as_float(q[r][j][e]), part[r][e], 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < RT; r++) sc[r][x] = (part[r][0] + part[r][1]) + (part[r][2] + part[r][3]);
                }
#pragma unroll
                for (int j = 0; j < (TYPE == kF32 ? 0 : C::NKL); j++) {
                    if constexpr (Q8) {
                        unsigned w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            w[e] = code_pair(kr[x][j][e >> 1], kr[x][j][e >> 1], e & 1 ? 0x0c030c02u : 0x0c010c00u);
                        const u4 kf = {w[0], w[1], w[2], w[3]};
                        const f4 f = *reinterpret_cast<const f4 *>(&k_scale[wave][j][16 * x + 4 * g]);
#pragma unroll
                        for (int r = 0; r < RT; r++) sc[r][x] += f * mfma16<kF16>(kf, q[r][j], f4{0, 0, 0, 0});
                    } else {
                        const u4 kf = {kr[x][j][0], kr[x][j][1], kr[x][j][2], kr[x][j][3]};
#pragma unroll
                        for (int r = 0; r < RT; r++) sc[r][x] = mfma16<C::MT>(kf, q[r][j], sc[r][x]);
                    }
                }
            }
            // scale, bias, masks: a key that a row does not see has -inf
            const f4 tile_bias[2] = {bias[0], bias[1]};
            if (t + 4 < t_hi) load_k(t + 4, next);
#pragma unroll
            for (int r = 0; r < RT; r++) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float v = sc[r][x][i] * to_score[r];
                        if constexpr (Q8 && QT == kBF16) v *= rest[r];
                        if (a.bias) v = SPECIAL && tile_bias[x][i] == -INFINITY ? -INFINITY : v + tile_bias[x][i];
                        sc[r][x][i] = v;
                    }
                if constexpr (SPECIAL) {
                    unsigned see = seen32(a, sq, tok[r], key0);
                    see &= (ok[0] ? 0xffffu : 0u) | (ok[1] ? 0xffff0000u : 0u);
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (!(see >> (16 * x + 4 * g + i) & 1)) sc[r][x][i] = -INFINITY;
                }
            }
            // running maximum and sum
            float ref[RT];
#pragma unroll
            for (int r = 0; r < RT; r++) {
                float t0 = fmaxf(fmaxf(sc[r][0][0], sc[r][0][1]), fmaxf(sc[r][0][2], sc[r][0][3]));
                float t1 = fmaxf(fmaxf(sc[r][1][0], sc[r][1][1]), fmaxf(sc[r][1][2], sc[r][1][3]));
                const float now = row_max(fmaxf(t0, t1));
                // (weights up to e^3 are left to grow before the sums are scaled)
                if (__ballot(now - mx[r] > 3.0f)) {
                    const float to = fmaxf(mx[r], now);
                    const float f = exp_of(mx[r] - (to == -INFINITY ? 0.0f : to));
                    mx[r] = to;
                    sum[r] *= f;
#pragma unroll
                    for (int c = 0; c < C::NC; c++) acc[r][c] *= f;
                }
                ref[r] = (mx[r] == -INFINITY ? 0.0f : mx[r]) - C::log_lift;
            }
            // V of keys that no row may see is not to be multiplied, whatever it holds; and where some
            // rows see a key and others do not, a value that is not finite reaches only those that do
            if constexpr (SPECIAL && !Q8) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int kk = 4 * x + i;
                        const bool there = key0 + 16 * x + 4 * g + i < held && ok[x];
#pragma unroll
                        for (int w = 0; w < C::NU; w++)
#pragma unroll
                            for (int y = 0; y < C::WV; y++) {
                                unsigned & z = vr[kk][w][y];
                                if (!there) z = 0;
                                if constexpr (TYPE == kF32) {
                                    if ((z & 0x7f800000u) == 0x7f800000u) {
                                        odd = true;
                                        z = 0;
                                    }
                                } else {
                                    constexpr unsigned e = TYPE == kF16 ? 0x7c00u : 0x7f80u;
                                    odd |= (z & e) == e || (z >> 16 & e) == e;
                                    if ((z & e) == e) z &= 0xffff0000u;
                                    if ((z >> 16 & e) == e) z &= 0xffffu;
                                }
                            }
                    }
            }
            // weights, as the second product's operand
            float p[RT][8];
#pragma unroll
            for (int r = 0; r < RT; r++) {
                float t = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    p[r][i] = exp_of(sc[r][i >> 2][i & 3] - ref[r]);
                    t += p[r][i];
                }
                sum[r] += t;
            }
            // O^T += V^T P^T
            if constexpr (TYPE == kF32) {
#pragma unroll
                for (int kk = 0; kk < 8; kk++)
#pragma unroll
                    for (int c = 0; c < C::NC; c++)
#pragma unroll
                        for (int r = 0; r < RT; r++)
                            acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(vr[kk][c / C::VW][c % C::VW]), p[r][kk], acc[r][c], 0, 0, 0);
            } else {
                u4 pf[RT];
#pragma unroll
                for (int r = 0; r < RT; r++)
                    pf[r] = u4{pack2<C::MT>(p[r][0], p[r][1]), pack2<C::MT>(p[r][2], p[r][3]), pack2<C::MT>(p[r][4], p[r][5]),
                               pack2<C::MT>(p[r][6], p[r][7])};
                if constexpr (Q8) {
                    if constexpr (SPECIAL) {
#pragma unroll
                        for (int kk = 0; kk < 8; kk++)
#pragma unroll
                            for (int c = 0; c < C::NC; c++) {
                                const float v = (float)v_scale[wave][C::column(m, c) / 32][16 * (kk >> 2) + 4 * g + (kk & 3)] *
                                                byte_value(vr[kk][c / C::VW], c % C::VW);
#pragma unroll
                                for (int r = 0; r < RT; r++)
                                    acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[r][kk], acc[r][c], 0, 0, 0);
                            }
                    } else {
                        h2 vs[4];
#pragma unroll
                        for (int c = 0; c < C::NC; c++) {
                            const int w = c / C::VW, y = c % C::VW;
                            if (y == 0) {
                                const _Float16 * f = &v_scale[wave][C::column(m, c) / 32][4 * g];
#pragma unroll
                                for (int e = 0; e < 4; e++) vs[e] = *reinterpret_cast<const h2 *>(f + 16 * (e >> 1) + 2 * (e & 1));
                            }
                            u4 vh, vl;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const h2 code = __builtin_bit_cast(h2, code_pair(vr[2 * e + 1][w][y >> 2], vr[2 * e][w][y >> 2],
                                                                                 0x0c040c00u + 0x00010001u * (y & 3)));
                                const h2 v = code * vs[e];
                                vh[e] = __builtin_bit_cast(unsigned, v);
                                if constexpr (QT == kF16)
                                    vl[e] = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(code, vs[e], -v));
                            }
#pragma unroll
                            for (int r = 0; r < RT; r++) {
                                acc[r][c] = mfma16<kF16>(vh, pf[r], acc[r][c]);
                                if constexpr (QT == kF16) acc[r][c] = mfma16<kF16>(vl, pf[r], acc[r][c]);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < C::NC; c++) {
                        const int w = c / C::VW, y = c % C::VW;
                        unsigned f[4];
#pragma unroll
                        for (int e = 0; e < 4; e++)   // halves y of keys 2e, 2e+1
                            f[e] = __builtin_amdgcn_perm(vr[2 * e + 1][w][y >> 1], vr[2 * e][w][y >> 1],
                                                         y & 1 ? 0x07060302u : 0x05040100u);
                        const u4 vf = {f[0], f[1], f[2], f[3]};
#pragma unroll
                        for (int r = 0; r < RT; r++) acc[r][c] = mfma16<C::MT>(vf, pf[r], acc[r][c]);
                    }
                }
            }
            if (SPECIAL && __ballot(odd)) odd_tiles.add(t);
            if (t + 4 < t_hi) load_v(t + 4, next);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                page[x] = next[x];
                next[x] = later[x];
            }
        };
        for (int t = t_lo + wave; t < t_hi;) {
            for (; t < t_hi && !special(t); t += 4) step(t, std::false_type{});
            for (; t < t_hi && special(t); t += 4) step(t, std::true_type{});
        }

        // the four waves' parts, and the result
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const float l = row_sum(sum[r]);
            const int row = 16 * r + m;
            if (g == 0) {
                join_m[wave][row] = mx[r];
                join_l[wave][row] = l;
            }
#pragma unroll
            for (int w = 0; w < C::NU; w++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int y = 0; y < C::VW; y += 4)
                        *reinterpret_cast<f4 *>(&join[wave][row][C::column(4 * g + i, w * C::VW + y)]) =
                            f4{acc[r][w * C::VW + y][i], acc[r][w * C::VW + y + 1][i], acc[r][w * C::VW + y + 2][i],
                               acc[r][w * C::VW + y + 3][i]};
        }
        if (lane == 0) join_odd[wave] = odd_tiles.bits;
        __syncthreads();
        for (int w = 0; w < 4; w++) odd_tiles.bits |= join_odd[w];
        for (int e = threadIdx.x; e < ROWS * (D / 4); e += 256) {
            const int r = e / (D / 4), col = e % (D / 4) * 4;
            const int row = row0 + r;
            if (row >= rows || col >= a.dv) continue;
            float top = join_m[0][r];
            for (int w = 1; w < 4; w++) top = fmaxf(top, join_m[w][r]);
            const float zero = top == -INFINITY ? 0.0f : top;
            f4 x = {0, 0, 0, 0};
            float l = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = exp_of(join_m[w][r] - zero) * (1.0f / C::lift);
                l += f * join_l[w][r];
                x += f * *reinterpret_cast<const f4 *>(&join[w][r][col]);
            }
            if (__builtin_expect(odd_tiles.bits != 0, 0)) {
                // what was left out reaches the rows that see its key
                Odd<TYPE, QT> o{a, sq, h, row / a.G, row % a.G};
                odd_tiles.each(32, held, [&](int key, int end) {
#pragma nounroll
                    for (; key < end; key++)
#pragma nounroll
                        for (int y = 0; y < 4 && col + y < a.dv; y++) {
                            const float add = o.term(key, col + y, zero);
                            x[0] += y == 0 ? add : 0.0f;
                            x[1] += y == 1 ? add : 0.0f;
                            x[2] += y == 2 ? add : 0.0f;
                            x[3] += y == 3 ? add : 0.0f;
                        }
                });
            }
            const long long out = (long long)(tok0 + row / a.G) * a.H * a.G + h * a.G + row % a.G;
            if (a.splits > 1) {
                const long long at = (long long)split * a.n_tok * a.H * a.G + out;
                for (int y = 0; y < 4 && col + y < a.dv && t_lo < t_hi; y++) a.part_o[at * a.dv + col + y] = x[y];
                if (col == 0) {
                    a.part_ml[2 * at] = top;
                    a.part_ml[2 * at + 1] = l;
                }
            } else {
                // (a row that sees a cell has a weight of 1 in its sum, or NaN)
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                char * o = a.o + ((long long)(tok0 + row / a.G) * a.o_tok + (long long)(h * a.G + row % a.G) * a.o_head) * C::ES;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    if (col + y >= a.dv) break;
                    const float v = x[y] * inv;
                    if constexpr (TYPE == kF32)
                        reinterpret_cast<float *>(o)[col + y] = v;
                    else
                        reinterpret_cast<unsigned short *>(o)[col + y] = (unsigned short)pack2<QT>(v, v);
                }
                if (a.lse && col == 0) a.lse[out] = l == 0.0f ? -INFINITY : top + logf(l);
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Many rows: 32 of them a wave, RW waves of rows (32 RW rows a block), over
// tiles of 64 keys that all waves read from LDS. KW = 2: half of the waves
// take the first 32 keys of each tile, half the others, and they join at the
// end (over a cache); or, PAIR, they swap their weights through LDS in every
// tile, and each sums half of the columns (prompts of heads wider than 128).
//
// Fragments (32x32x16, lane l, n = l % 32, h = l / 32): an operand's lane holds
// row n and elements 8h .. 8h+7 of the summed axis; a result's lane column n
// and rows 8x + 4h + y (register 4x + y). As in k_attn_rows the scores of one
// row of the caller's are one lane's (two lanes', h = 0 and 1), and go into the
// second product from the registers they were made in: element j of step s is
// key 16s + 4h + j, or 16s + 8 + 4h + j - 4.
//
// K and V reach LDS by direct loads of 16 bytes a lane (no registers), a
// uniform address and a lane's constant offset each. They stand row by row with
// their 16-byte pieces exchanged, K's by key % 8 so that the rows of a fragment
// read different banks, V's in pairs by key % 8 so that the four rows that
// ds_read_b64_tr_b16 turns round do: it gives a lane four keys of one column,
// half a fragment of V^T. Pieces past a head's width stay zero.
//
// A prompt's blocks are four waves, two of them on a CU: one's softmax runs
// under the other's products, and K and V come from L2 (one tile ahead). They
// are bound by what issues beside the products: 16384 tokens of 32 heads of 128
// take 2.2 to 2.34 ms by card, 940 to 995 TFLOP/s (a large matrix product: 1130;
// 4 % more with one loop for plain and masked tiles; matrix units busy 46 % of
// the cycles, vector instructions 44 %), 12 prompts of as many in all 0.56 to
// 0.59 ms (37 % and 43 %: the last blocks of ragged prompts).
// At 256 columns a wave's sums and queries alone are 192 registers, which
// leaves one wave a SIMD and a third of its instructions moves between the
// halves of the file: 5003 tokens in three prompts of 8 heads took 132 us that
// way and take 89 us in pairs (128 + 16 KB of LDS, one block a CU; bound by the
// longest prompt's chain of tiles, which three barriers a tile stretch).
//
// Over a cache HBM has to be kept busy: eight waves share four buffers (RW = 4:
// 96 KB on their way), or two blocks of four waves two buffers each (RW = 2).
// Eight sequences of up to 20000 F16 cells, 8 x 128, with 32 drafts of 32 heads
// take 157 us, 2.7 TB/s (163 with one loop for plain and masked tiles); bound by
// the last blocks of ragged sequences and by a step's latency, 2.2 us where its
// loads alone would take 1.7 (matrix units busy 14 %, vector instructions 27 %).
__device__ const unsigned zero_word = 0;
__device__ const unsigned hidden_word = 0xff800000u;   // -inf

typedef float f16x __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

template <int TYPE> __device__ __forceinline__ f16x mfma32(u4 a, u4 b, f16x c) {
    if constexpr (TYPE == kF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float pair_max(float x) { return fmaxf(x, __shfl_xor(x, 32)); }

// KW: halves of a tile's keys that waves share out
constexpr int tile_halves(bool cells, int d) { return cells || d == 256 ? 2 : 1; }

template <int TYPE, int D, bool CELLS, int RW>
__global__ __launch_bounds__(64 * RW * tile_halves(CELLS, D), CELLS && D == 256 ? 1 : 2)
void k_attn_tiles(AttnArgs a) {
    constexpr bool PAIR = !CELLS && D == 256;               // two waves share their rows' weights, and halve the columns
    constexpr int KW = tile_halves(CELLS, D), WAVES = RW * KW, ROWS = 32 * RW;
    constexpr int BK = 64, SUB = BK / 32 / KW;              // keys of a tile; of a wave's scores, in parts of 32
    constexpr int KS = D / 16, DT = D / 32 / (PAIR ? 2 : 1), CH = D / 8;   // steps of a score, column tiles, pieces of a row
    constexpr int PV = PAIR ? 2 : SUB;                      // parts of 32 keys in a wave's second product
    constexpr int NL = BK * CH / (64 * WAVES);              // direct loads of a wave and tile, K or V
    constexpr int KPL = 512 / D;                            // keys of one: rows of one 16-cell group
    constexpr int BUFS = CELLS && RW == 4 && D < 256 ? 4 : 2, AHEAD = BUFS - 1;
    constexpr int ROWB = 2 * D, VX = CH < 16 ? CH / 2 - 1 : 7;
    constexpr int LOADS = 2 * NL + (CELLS ? 1 : 0);         // of a wave and tile
    constexpr float lift = TYPE == kF16 ? 0x1p10f : 1.0f, log2_lift = TYPE == kF16 ? 10.0f : 0.0f;
    __shared__ __align__(16) char lds[BUFS][2][BK * ROWB];  // [buffer][K, V]
    static_assert(KW == 1 || PAIR || RW * (DT * 4 + 1) * 64 * 16 <= BUFS * 2 * BK * ROWB, "parts handed over fit the tiles");
    __shared__ __align__(16) u4 swap[PAIR ? WAVES : 1][2][64];     // a wave's weights, lane for lane
    __shared__ float swap_top[PAIR ? WAVES : 1][64];
    __shared__ __align__(16) float cells[BUFS][CELLS ? BK : 1];   // bias of each cell; -inf: hidden from every row

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rw = wave % RW, kw = wave / RW;
    const int n = lane & 31, hf = lane >> 5;
    const int other = PAIR ? rw + RW * (1 - kw) : 0;         // the wave of the same rows
    const int d0 = PAIR ? DT * kw : 0;                       // column tiles: this one and DT - 1 more
    auto meet = [] {   // (direct loads stay on their way)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    int u = blockIdx.x;
    const int h = u % a.H;
    u /= a.H;
    int split = 0;
    if constexpr (CELLS) {
        split = u % a.splits;
        u /= a.splits;
    }
    int s, tile, tile_step;
    if (CELLS && a.tiles) {
        tile = u % a.tiles;
        s = u / a.tiles;
        tile_step = a.tiles;
    } else {
        if (!find_tile(a, u, ROWS, lane, s, tile)) return;
        tile_step = 1 << 30;
    }
    s = __builtin_amdgcn_readfirstlane(s);
    tile = __builtin_amdgcn_readfirstlane(tile);
    const Sequence q = sequence_of(a, s);
    if (q.n_new <= 0) return;
    const int rows = q.n_new * a.G;
    const int page_mask = CELLS ? (1 << a.shift) - 1 : 0;
    const bool flip = a.scale < 0.0f;   // (the maximum is taken of products by a positive number)
    const float scale = fabsf(a.scale);
    const float c = (CELLS ? 1.0f : scale) * kLog2e;   // (CELLS: scores take the scale with the bias)

    // A lane's piece of a direct load: its row there, and where that stands.
    // (The exchange of pieces is the same in all of a wave's loads.)
    const int piece_row = lane / CH, piece_key = wave * KPL + piece_row;
    const unsigned k_col = (lane % CH) ^ (piece_key & 7), v_col = (lane % CH) ^ ((piece_key & VX) << 1);
    const unsigned k_off = __umul24(piece_row, a.k.ld_tok) + 16 * k_col, v_off = __umul24(piece_row, a.v.ld_tok) + 16 * v_col;
    const bool k_piece = (int)(8 * k_col) < a.dk, v_piece = (int)(8 * v_col) < a.dv;
    const char * k_head = a.k.base + h * a.k.ld_head;
    const char * v_head = a.v.base + h * a.v.ld_head;
    for (int i = threadIdx.x; i < BUFS * 2 * BK * CH; i += 64 * WAVES) reinterpret_cast<u4 *>(lds)[i] = u4{0, 0, 0, 0};
    __syncthreads();

    for (; (long long)tile * ROWS < rows; tile += tile_step) {
        const int row0 = tile * ROWS, wrow0 = row0 + 32 * rw;
        const int last_tok = (row0 + ROWS - 1) / a.G < q.n_new ? (row0 + ROWS - 1) / a.G : q.n_new - 1;
        const int end_all = q.held == 0 ? 0 : (CELLS && a.mask ? q.held : q.base + last_tok + 1);
        // keys before it are seen by every row of this wave
        const int clear = CELLS && a.mask ? q.base : q.base + (wrow0 < rows ? wrow0 / a.G + 1 : last_tok + 1);
        const int n_tiles = (end_all + BK - 1) / BK;
        int t_lo = 0, t_hi = n_tiles;
        if constexpr (CELLS) {
            const int per = range_tiles(a, n_tiles, BK);
            t_lo = split * per;
            t_hi = t_lo + per < n_tiles ? t_lo + per : n_tiles;
        }
        const int row = wrow0 + n;
        const bool on = row < rows;
        const int tok = on ? row / a.G : 0, head = on ? row % a.G : 0;
        u4 qf[KS];
        {
            const char * p = a.q + 2 * ((long long)(q.tok0 + tok) * a.q_tok + (long long)(h * a.G + head) * a.q_head);
#pragma unroll
            for (int j = 0; j < KS; j++) {
                qf[j] = 16 * j + 8 * hf < a.dk ? *reinterpret_cast<const u4 *>(p + 32 * j + 16 * hf) : u4{0, 0, 0, 0};
                if (flip) qf[j] ^= 0x80008000u;
            }
        }

        // pages of a tile's pieces, and of the 16 cells whose biases this wave loads
        int page[CELLS ? NL + 1 : 1];
        auto page_at = [&](int key) { return key < end_all ? uniform_load(q.table + (key >> a.shift)) : -1; };
        auto find_pages = [&](int t) {
            if constexpr (CELLS) {
#pragma unroll
                for (int i = 0; i < NL; i++) page[i] = page_at(t * BK + (i * WAVES + wave) * KPL);
                page[NL] = page_at(t * BK + 16 * (wave % (BK / 16)));
            }
        };
        // (Rows of a page past the last cell are loaded as they are, those of a
        // bad page from page 0: their cells are hidden. Rows past the end of
        // contiguous tokens are not loaded. A tile past the last one is loaded
        // like the last, so that every wave has the same loads on their way.)
        auto fill = [&](int t, int buf) {
            if (t >= t_hi) t = t_hi - 1;
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int key = t * BK + (i * WAVES + wave) * KPL;
                unsigned at;
                bool there = true;
                if constexpr (CELLS) {
                    const int p = page[i] >= 0 && page[i] < a.n_pages ? page[i] : 0;
                    at = ((unsigned)p << a.shift) + (key & page_mask);
                } else {
                    at = (unsigned)(q.tok0 + key);
                    there = key + piece_row < q.held;
                }
                char * to = &lds[buf][0][(i * WAVES + wave) * 1024];
                if (there && k_piece) load_lds16(k_head + (unsigned long long)at * a.k.ld_tok, k_off, to);
                if (there && v_piece) load_lds16(v_head + (unsigned long long)at * a.v.ld_tok, v_off, to + BK * ROWB);
            }
            if constexpr (CELLS) {
                const int in = 16 * (wave % (BK / 16)), key = t * BK + in + (lane & 15);
                const char * b = reinterpret_cast<const char *>(&hidden_word);
                if (key < end_all && page[NL] >= 0 && page[NL] < a.n_pages)
                    b = a.bias ? reinterpret_cast<const char *>(a.bias + (((long long)page[NL] * a.H + h) << a.shift) + (key & page_mask))
                               : reinterpret_cast<const char *>(&zero_word);
                if (lane < 16) load_lds4(b, reinterpret_cast<char *>(&cells[buf][in]));
            }
        };

        f16x acc[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
        OddTiles odd_tiles(t_lo, t_hi);     // with values that are not finite and were left out (see below)
        float mx = -INFINITY, sum = 0.0f;   // (mx: in units of s, kept up to 2^5 below the true maximum)
        float mc = 0.0f;                    // mx, or 0 while nothing is seen

        if (t_lo < t_hi) {
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                find_pages(t_lo + i < t_hi ? t_lo + i : t_hi - 1);
                fill(t_lo + i, i);
            }
            find_pages(t_lo + AHEAD < t_hi ? t_lo + AHEAD : t_hi - 1);
        }
        // until tile t is there; the next loads go
        auto arrive = [&](int t) {
            wait_lds_loads<(AHEAD - 1) * LOADS>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            fill(t + AHEAD, (t - t_lo + AHEAD) % BUFS);
            find_pages(t + AHEAD + 1 < t_hi ? t + AHEAD + 1 : t_hi - 1);
        };
        // PLAIN: no key of the wave's part of the tile is hidden from one of its rows (!CELLS: of the block's)
        auto step = [&](int t, auto kind) {
            constexpr bool PLAIN = decltype(kind)::value;
            const int buf = (t - t_lo) % BUFS;
            const int part0 = 32 * SUB * kw, key0 = t * BK + part0;   // this wave's keys of the tile
            const char * kt = lds[buf][0] + part0 * ROWB;
            const char * vt = lds[buf][1] + (PAIR ? 0 : part0 * ROWB);

            f16x sc[SUB];
#pragma unroll
            for (int x = 0; x < SUB; x++) {
#pragma unroll
                for (int i = 0; i < 16; i++) sc[x][i] = 0.0f;
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    const u4 kf = *reinterpret_cast<const u4 *>(kt + (32 * x + n) * ROWB + (((2 * j + hf) ^ (n & 7)) << 4));
                    sc[x] = mfma32<TYPE>(kf, qf[j], sc[x]);
                }
            }
            bool hidden = false;   // (uniform) a key that some row does not see
            if constexpr (CELLS) {
                hidden = !PLAIN;
#pragma unroll
                for (int x = 0; x < SUB; x++)
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const f4 b = *reinterpret_cast<const f4 *>(&cells[buf][part0 + 32 * x + 8 * y + 4 * hf]);
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[x][4 * y + i] = sc[x][4 * y + i] * scale + b[i];
                    }
                if (!PLAIN) {   // (whatever the product was)
#pragma unroll
                    for (int x = 0; x < SUB; x++)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (cells[buf][part0 + 32 * x + 8 * (i >> 2) + 4 * hf + (i & 3)] == -INFINITY) sc[x][i] = -INFINITY;
                }
            }
            if (!PLAIN && key0 + 32 * SUB > clear) {
#pragma unroll
                for (int x = 0; x < SUB; x++) {
                    const unsigned see = seen32(a, q, tok, key0 + 32 * x) >> (4 * hf);
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (!(see >> (8 * (i >> 2) + (i & 3)) & 1)) sc[x][i] = -INFINITY;
                }
                hidden = true;
            }

            float top = sc[0][0];
#pragma unroll
            for (int x = 0; x < SUB; x++)
#pragma unroll
                for (int i = 0; i < 16; i++) top = fmaxf(top, sc[x][i]);
            top = pair_max(top);
            if constexpr (PAIR) {
                swap_top[wave][lane] = top;
                meet();
                top = fmaxf(top, swap_top[other][lane]);
                hidden = !PLAIN && t * BK + BK > clear;   // (V of both halves)
            }
            // weights up to 2^5 are left to grow before the sums are scaled
            if (__ballot((top - mx) * c > 5.0f)) {
                const float now = fmaxf(mx, top);
                const float use = now == -INFINITY ? 0.0f : now;
                const float f = __builtin_amdgcn_exp2f((mx - use) * c);
                mx = now;
                mc = use;
                sum *= f;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[d][i] *= f;
            }
            // weights, and V
            float p[SUB][16];
            float part = 0.0f;
            const float off = log2_lift - mc * c;
#pragma unroll
            for (int x = 0; x < SUB; x++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    // (with a bias the difference first: a score may be the type's lowest value)
                    p[x][i] = CELLS ? __builtin_amdgcn_exp2f((sc[x][i] - mc) * c + log2_lift)
                                    : __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][i], c, off));
                    part += p[x][i];
                }
            sum += part;
            u4 pf[PV][2];
#pragma unroll
            for (int x = 0; x < SUB; x++)
#pragma unroll
                for (int st = 0; st < 2; st++)
#pragma unroll
                    for (int e = 0; e < 4; e++) pf[x][st][e] = pack2<TYPE>(p[x][8 * st + 2 * e], p[x][8 * st + 2 * e + 1]);
            if constexpr (PAIR) {   // (the wave's own part first, then the other's)
                swap[wave][0][lane] = pf[0][0];
                swap[wave][1][lane] = pf[0][1];
                meet();
                pf[1][0] = swap[other][0][lane];
                pf[1][1] = swap[other][1][lane];
            }
            bool odd = false;
#pragma unroll
            for (int x0 = 0; x0 < PV; x0++)
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    const int x = PAIR ? x0 ^ kw : x0;
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        u2 half[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int r = (lane & 15) >> 2;   // key 4 hf + r of the eight
                            const int col = 4 * (d0 + d) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                            const char * at = vt + (32 * x + 16 * st + 8 * e + 4 * hf + r) * ROWB +
                                              ((col ^ (((4 * hf + r) & VX) << 1)) << 4) + ((lane & 1) << 3);
                            half[e] = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                                 (__attribute__((address_space(3))) s4 *)at));
                        }
                        u4 vf = {half[0].x, half[0].y, half[1].x, half[1].y};
                        if (!PLAIN && hidden) {
                            constexpr unsigned e = TYPE == kF16 ? 0x7c00u : 0x7f80u;
#pragma unroll
                            for (int y = 0; y < 4; y++) {
                                const bool lo = (vf[y] & e) == e, hi = (vf[y] >> 16 & e) == e;
                                // (cells that no row sees, past the end among them, are nothing)
                                const int kk = 32 * x + 16 * st + 8 * (y >> 1) + 4 * hf + 2 * (y & 1);
                                if (lo) odd |= CELLS ? cells[buf][part0 + kk] != -INFINITY : (PAIR ? t * BK : key0) + kk < q.held;
                                if (hi) odd |= CELLS ? cells[buf][part0 + kk + 1] != -INFINITY : (PAIR ? t * BK : key0) + kk + 1 < q.held;
                                vf[y] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                            }
                        }
                        acc[d] = mfma32<TYPE>(vf, pf[x0][st], acc[d]);
                    }
                }
            if (!PLAIN && hidden && __ballot(odd)) odd_tiles.add(t);
        };
        // (Loops apart for the two kinds: a branch around each product would keep
        // it behind its own load of V, two copies of the products in one loop
        // would each want sums of their own.)
        int t = t_lo;
        if constexpr (CELLS) {
            auto whole = [&](int t) {
                const int part0 = 32 * SUB * kw;
                return t * BK + part0 + 32 * SUB <= clear &&
                       __ballot(cells[(t - t_lo) % BUFS][part0 + (lane & (32 * SUB - 1))] == -INFINITY) == 0;
            };
            bool plain = false;
            if (t < t_hi) {
                arrive(t);
                plain = whole(t);
            }
            while (t < t_hi) {
                while (t < t_hi && plain) {
                    step(t, std::true_type{});
                    if (++t < t_hi) {
                        arrive(t);
                        plain = whole(t);
                    }
                }
                while (t < t_hi && !plain) {
                    step(t, std::false_type{});
                    if (++t < t_hi) {
                        arrive(t);
                        plain = whole(t);
                    }
                }
            }
        } else {
            const int plain = min((q.base + row0 / a.G + 1) / BK, t_hi);
            for (; t < plain; t++) {
                arrive(t);
                step(t, std::true_type{});
            }
            for (; t < t_hi; t++) {
                arrive(t);
                step(t, std::false_type{});
            }
        }
        wait_lds_loads<0>();   // (LDS is given up, or used again, with no load to it on its way)
        sum += __shfl_xor(sum, 32);
        if constexpr (PAIR) {
            swap_top[wave][lane] = sum;
            __syncthreads();
            sum = kw ? swap_top[other][lane] + sum : sum + swap_top[other][lane];
        } else if constexpr (KW == 2) {
            // the second half of the waves hands its part over, lane for lane
            f4 * over = reinterpret_cast<f4 *>(lds) + rw * (DT * 4 + 1) * 64 + lane;
            __syncthreads();
            if (kw == 1) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        over[(4 * d + y) * 64] = f4{acc[d][4 * y], acc[d][4 * y + 1], acc[d][4 * y + 2], acc[d][4 * y + 3]};
                over[DT * 4 * 64] = f4{mx, sum, __uint_as_float((unsigned)odd_tiles.bits), __uint_as_float((unsigned)(odd_tiles.bits >> 32))};
            }
            __syncthreads();
            if (kw == 0) {
                const f4 theirs = over[DT * 4 * 64];
                const float top = fmaxf(mx, theirs[0]), use = top == -INFINITY ? 0.0f : top;
                const float f = __builtin_amdgcn_exp2f((mx - use) * c), g = __builtin_amdgcn_exp2f((theirs[0] - use) * c);
                mx = top;
                sum = sum * f + theirs[1] * g;
                odd_tiles.bits |= __float_as_uint(theirs[2]) | (unsigned long long)__float_as_uint(theirs[3]) << 32;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const f4 x = over[(4 * d + y) * 64];
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[d][4 * y + i] = acc[d][4 * y + i] * f + x[i] * g;
                    }
            }
        }
        sum *= 1.0f / lift;
        const long long out = (long long)(q.tok0 + tok) * a.H * a.G + h * a.G + head;
        const bool write = on && (PAIR || kw == 0);
        if (CELLS && a.splits > 1) {
            const long long at = (long long)split * a.n_tok * a.H * a.G + out;
            if (write) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const int col = 32 * (d0 + d) + 8 * y + 4 * hf;
                        if (col < a.dv && t_lo < t_hi)
                            *reinterpret_cast<f4 *>(a.part_o + at * a.dv + col) =
                                f4{acc[d][4 * y], acc[d][4 * y + 1], acc[d][4 * y + 2], acc[d][4 * y + 3]} * (1.0f / lift);
                    }
                if (hf == 0) {
                    a.part_ml[2 * at] = CELLS ? mx : mx * scale;
                    a.part_ml[2 * at + 1] = sum;
                }
            }
        } else if (write) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / (sum * lift);
            char * o = a.o + 2 * ((long long)(q.tok0 + tok) * a.o_tok + (long long)(h * a.G + head) * a.o_head);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const int col = 32 * (d0 + d) + 8 * y + 4 * hf;
                    if (col >= a.dv) continue;
                    const u2 v = {pack2<TYPE>(acc[d][4 * y] * inv, acc[d][4 * y + 1] * inv),
                                  pack2<TYPE>(acc[d][4 * y + 2] * inv, acc[d][4 * y + 3] * inv)};
                    *reinterpret_cast<u2 *>(o + 2 * col) = v;
                }
            if (a.lse && hf == 0 && kw == 0)
                a.lse[out] = sum == 0.0f ? -INFINITY : (CELLS ? mx : mx * scale) + logf(sum);
        }
        if (__builtin_expect(odd_tiles.bits != 0, 0) && write && sum == sum) {
            // Values that are not finite were left out of tiles where a key is
            // hidden from some row. They decide every result they reach (of rows
            // that are not NaN by their scores): those are written again.
            Odd<TYPE, TYPE> o{a, q, h, tok, head};
            const float top = (mx == -INFINITY ? 0.0f : mx) * (CELLS ? 1.0f : scale);
#pragma nounroll
            for (int col = 32 * d0 + hf; col < a.dv && col < 32 * (d0 + DT); col += 2) {
                float x = 0.0f;
                odd_tiles.each(BK, q.held, [&](int key, int end) {
#pragma nounroll
                    for (; key < end; key++) x += o.term(key, col, top);
                });
                if (x == 0.0f) continue;
                if (CELLS && a.splits > 1)
                    a.part_o[((long long)split * a.n_tok * a.H * a.G + out) * a.dv + col] = x;
                else
                    reinterpret_cast<unsigned short *>(a.o)[(long long)(q.tok0 + tok) * a.o_tok +
                                                            (long long)(h * a.G + head) * a.o_head + col] =
                        (unsigned short)pack2<TYPE>(x, x);
            }
        }
        __syncthreads();
        if (KW == 2 && !PAIR && (long long)(tile + tile_step) * ROWS < rows) {
            // (what was handed over stood on pieces that are to be zero)
            for (int i = threadIdx.x; i < BUFS * 2 * BK * CH; i += 64 * WAVES) reinterpret_cast<u4 *>(lds)[i] = u4{0, 0, 0, 0};
            __syncthreads();
        }
    }
}

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

int head_tile(int dk, int dv) {
    const int d = dk > dv ? dk : dv;
    return d <= 64 ? 64 : d <= 128 ? 128 : 256;
}

bool vec_rows(const kvc_heads & x, int bytes) {
    return ((reinterpret_cast<uintptr_t>(x.data) | (uintptr_t)(x.ld_tok * bytes) | (uintptr_t)(x.ld_head * bytes)) & 15) == 0;
}

template <int TYPE, int QT, int D, int RT, Columns COLS> bool run_rows(const AttnArgs & a, long long blocks, hipStream_t st) {
    return launch(k_attn_rows<TYPE, QT, D, RT, COLS>, dim3((unsigned)blocks), dim3(256), st, a);
}
template <int TYPE, int QT, int D> bool run_rows(const AttnArgs & a, int rt, bool careful, long long blocks, hipStream_t st) {
    if constexpr (TYPE != kQ8)
        if (careful) return run_rows<TYPE, QT, D, 1, ANY>(a, blocks, st);
    const bool full = a.dk == D && a.dv == D;
    if constexpr (TYPE == kQ8 && D < 256)
        if (rt == 4) return full ? run_rows<TYPE, QT, D, 4, FULL>(a, blocks, st) : run_rows<TYPE, QT, D, 4, PART>(a, blocks, st);
    if constexpr (D < 256)
        if (rt == 2) return full ? run_rows<TYPE, QT, D, 2, FULL>(a, blocks, st) : run_rows<TYPE, QT, D, 2, PART>(a, blocks, st);
    return full ? run_rows<TYPE, QT, D, 1, FULL>(a, blocks, st) : run_rows<TYPE, QT, D, 1, PART>(a, blocks, st);
}
template <int TYPE, int QT> bool run_rows(const AttnArgs & a, int d, int rt, bool careful, long long blocks, hipStream_t st) {
    if (d == 64) return run_rows<TYPE, QT, 64>(a, rt, careful, blocks, st);
    if (d == 128) return run_rows<TYPE, QT, 128>(a, rt, careful, blocks, st);
    return run_rows<TYPE, QT, 256>(a, rt, careful, blocks, st);
}
bool run_rows(const AttnArgs & a, int type, int qt, int rt, bool careful, long long blocks, hipStream_t st) {
    const int d = head_tile(a.dk, a.dv);
    if (type == kF32) return run_rows<kF32, kF32>(a, d, rt, careful, blocks, st);
    if (type == kF16) return run_rows<kF16, kF16>(a, d, rt, careful, blocks, st);
    if (type == kBF16) return run_rows<kBF16, kBF16>(a, d, rt, careful, blocks, st);
    if (qt == kF16) return run_rows<kQ8, kF16>(a, d, rt, careful, blocks, st);
    return run_rows<kQ8, kBF16>(a, d, rt, careful, blocks, st);
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

template <int TYPE, bool CELLS, int RW> bool run_tiles(const AttnArgs & a, int d, long long blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block(64 * RW * tile_halves(CELLS, d));
    if (d == 64) return launch(k_attn_tiles<TYPE, 64, CELLS, RW>, grid, block, st, a);
    if (d == 128) return launch(k_attn_tiles<TYPE, 128, CELLS, RW>, grid, block, st, a);
    if constexpr (CELLS && RW == 4) return false;   // (not asked for: eight waves' sums of 256 columns do not fit)
    else return launch(k_attn_tiles<TYPE, 256, CELLS, RW>, grid, block, st, a);
}
template <bool CELLS, int RW> bool run_tiles(const AttnArgs & a, int type, long long blocks, hipStream_t st) {
    const int d = head_tile(a.dk, a.dv);
    return type == kF16 ? run_tiles<kF16, CELLS, RW>(a, d, blocks, st) : run_tiles<kBF16, CELLS, RW>(a, d, blocks, st);
}

int esize(int type) { return type == kF32 ? 4 : 2; }

// Row numbers stay clear of 2^31 with a tile added, and a launch has fewer than
// 2^32 threads (blocks of 512 at most). (Key ranges only multiply launches of
// fewer than 4096 blocks, to less than twice that.)
constexpr long long kMaxRows = 1 << 30, kMaxBlocks = (1 << 23) - 1;

// Shape of a cache call's launch (n_seq > 0).
struct CacheShape {
    int rt, tiles, splits, range;
    bool careful;
    int whole;   // waves of rows of k_attn_tiles, 0: k_attn_rows
};
CacheShape cache_shape(const kvc_cache * c, const kvc_cache_attn_args * a) {
    CacheShape s{};
    const int G = a->n_head / c->n_head_kv, es = esize(a->type);
    // a cache's pages are 16-byte aligned: its rows are where a head is whole 16-byte pieces
    s.careful = c->k_type != kQ8 && (!vec_rows(a->q, es) || c->d_k * es % 16 || c->d_v * es % 16);
    const long long rows = (long long)a->max_new * G;
    s.rt = row_tiles(c->k_type, head_tile(c->d_k, c->d_v), s.careful, rows);
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
    const int max_len = a->max_len < 1 << 30 ? a->max_len : 1 << 30;   // (no sequence has more; sums with it stay in range)
    const long long units = (long long)a->n_seq * c->n_head_kv * s.tiles, blocks = s.whole || s.rt == 4 ? 1024 : 4096;
    long long want = (blocks + units - 1) / units, most = max_len / 256;
    want = want < most ? want : most;
    if ((long long)a->n_tok * a->n_head > 1 << 24) want = 1;   // (the join's launch: a block a row or four; so many need no ranges)
    s.splits = (int)(want < 1 ? 1 : want > 64 ? 64 : want);
    s.range = s.rt == 4 ? 0 : (max_len + s.splits - 1) / s.splits;
    return s;
}

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

}  // namespace

}  // namespace kvc

using namespace kvc;

extern "C" {

size_t kvc_attn_cache_workspace(const kvc_cache * c, const kvc_cache_attn_args * a) {
    if (check_cache_attn(c, a) || a->n_seq == 0 || a->n_tok == 0) return 0;
    const CacheShape s = cache_shape(c, a);
    return s.splits > 1 ? (size_t)s.splits * a->n_tok * a->n_head * (c->d_v + 2) * sizeof(float) : 0;
}

int kvc_attn_cache(const kvc_cache * c, const kvc_cache_attn_args * x, void * ws, size_t ws_bytes, void * stream) {
    if (int rc = check_cache_attn(c, x)) return rc;
    if (x->n_seq == 0 || x->n_tok == 0) return 0;
    if (!x->q.data || !x->o.data || !x->cu) return -1;
    const int es = esize(x->type);
    if ((reinterpret_cast<uintptr_t>(x->q.data) | reinterpret_cast<uintptr_t>(x->o.data)) & (es - 1))
        return KV_COMPACT_E_UNSUPPORTED;
    const CacheShape s = cache_shape(c, x);
    const size_t need = kvc_attn_cache_workspace(c, x);
    if (need && !ws) return -1;
    if (need && reinterpret_cast<uintptr_t>(ws) & 15) return KV_COMPACT_E_UNSUPPORTED;
    if (need > ws_bytes) return KVC_E_SCRATCH;
    const long long krow = (long long)kv_quant_row_bytes(c->k_type, c->n_head_kv * c->d_k);
    const long long vrow = (long long)kv_quant_row_bytes(c->v_type, c->n_head_kv * c->d_v);
    const long long cells = (long long)c->n_pages * c->page_size;
    if (krow >= 1 << 24 || vrow >= 1 << 24) return KV_COMPACT_E_UNSUPPORTED;
    AttnArgs a{};
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
    a.splits = s.splits; a.range = s.range; a.tiles = s.tiles;
    a.scale = x->scale != 0.0f ? x->scale : 1.0f / sqrtf((float)c->d_k);
    a.part_o = static_cast<float *>(ws);
    a.part_ml = a.part_o + (size_t)s.splits * x->n_tok * x->n_head * c->d_v;
    const long long blocks = (long long)x->n_seq * s.tiles * s.splits * a.H;
    if (blocks > kMaxBlocks) return KV_COMPACT_E_UNSUPPORTED;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    if (!(s.whole == 4   ? run_tiles<true, 4>(a, x->type, blocks, st)
          : s.whole == 2 ? run_tiles<true, 2>(a, x->type, blocks, st)
                         : run_rows(a, c->k_type, x->type, s.rt, s.careful, blocks, st)))
        return KV_COMPACT_E_DEVICE;
    if (s.splits > 1) {
        if (!(x->type == kF32 ? run_join<kF32>(a, st) : x->type == kF16 ? run_join<kF16>(a, st) : run_join<kBF16>(a, st)))
            return KV_COMPACT_E_DEVICE;
    }
    return 0;
}

int kvc_attn_prompt(const kvc_prompt_args * x, void * stream) {
    if (!x) return -1;
    if (x->n_seq < 0 || x->n_tok < 0 || x->n_head <= 0 || x->n_head_kv <= 0 || x->d_k <= 0 || x->d_v <= 0 ||
        x->n_head % x->n_head_kv)
        return -2;
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
    return (whole ? run_tiles<false, 4>(a, x->type, tiles * a.H, st)
                  : run_rows(a, x->type, x->type, rt, careful, tiles * a.H, st))
               ? 0
               : KV_COMPACT_E_DEVICE;
}

}  // extern "C"
