// k_weigh_rows over F32 cells (cut out of kvc_weigh.hip and kvc_attn_kernels.h
// by the test that builds this) on the CPU, lane by lane.
//
// stdin: int32 split, first wave to run, H, G, page size, pages, cells, tokens,
// first, last, cell tiles; float decay; table, q [tokens][H * G][64], k [page]
// [cell][H][64], lse [tokens][H * G], weights [H][cells in whole pages].
// stdout: the weights.
#include <algorithm>
#include <type_traits>

#include "block.h"

typedef float sums4 __attribute__((ext_vector_type(4)));
// D = A B + C of 16 x 16 results over 4: lane l has A[l % 16][l / 16], B[l / 16][l % 16] and D[4 (l / 16) + i][l % 16]
sums4 mfma_16x16x4(float a, float b, sums4 c) {
    const Post * p = gather(__float_as_uint(a), __float_as_uint(b));
    for (int i = 0; i < 4; i++)
        for (int k = 0; k < 4; k++)
            c[i] += __uint_as_float(p[16 * k + 4 * (lane_of() >> 4) + i].a) * __uint_as_float(p[16 * k + (lane_of() & 15)].b);
    return c;
}
using std::max;
template <class C> C no_product(C c) { exit(5); }

#define __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, ...) mfma_16x16x4(a, b, c)
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, ...) no_product(c)
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, ...) no_product(c)
#define __builtin_amdgcn_perm(a, b, pick) 0u
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_fence(order, scope)
#define __builtin_amdgcn_wave_barrier()
#define KV_TYPE_F32 0
#define KV_TYPE_F16 1
#define KV_TYPE_Q8_0 8
#define KV_TYPE_BF16 30
#include "weigh_rows.inc"

int main() {
    const std::vector<int> h = take<int>(11);
    const bool split = h[0];
    const int first = h[1], cells = h[6], tokens = h[7];
    WeighArgs w{};
    AttnArgs & a = w.a;
    a.H = h[2], a.G = h[3], a.shift = __builtin_ctz(h[4]), a.n_pages = h[5], a.first = h[8], a.last = h[9];
    w.cell_tiles = h[10];
    w.decay = take<float>(1)[0];
    a.max_pages = (cells + h[4] - 1) / h[4];
    w.room = a.max_pages * h[4];
    w.w_seq = a.H * w.room;
    const std::vector<int> table = take<int>(a.max_pages), cu = {0, tokens}, len = {cells};
    const std::vector<float> q = take<float>((size_t)tokens * a.H * a.G * 64), k = take<float>((size_t)a.n_pages * h[4] * a.H * 64);
    std::vector<float> lse = take<float>((size_t)tokens * a.H * a.G), weight = take<float>(w.w_seq);
    a.k = RowsAt{reinterpret_cast<const char *>(k.data()), 256, (unsigned)(256 * a.H)};
    a.q = reinterpret_cast<const char *>(q.data());
    a.q_tok = 64 * a.H * a.G, a.q_head = 64;
    a.lse = lse.data(), a.cu = cu.data(), a.len = len.data(), a.table = table.data();
    a.n_seq = a.max_seqs = 1, a.n_tok = tokens, a.dk = a.dv = 64, a.scale = 0.125f;
    w.weight = weight.data();
    for (blockIdx.x = 0; blockIdx.x < (unsigned)(a.H * w.cell_tiles); blockIdx.x++)
        run_block(4, first, [&] {
            if (split) k_weigh_rows<kF32, kF32, 64, kFewRows32, FULL, true>(w);
            else k_weigh_rows<kF32, kF32, 64, kFewRows32, FULL, false>(w);
        });
    give(weight);
    return 0;
}
