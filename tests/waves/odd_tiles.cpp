// Which keys the search for values that are not finite goes through under a
// window (KeyTiles and OddTiles, cut out of kvc_attn_kernels.h by the test that
// builds this).
//
// stdin, any number of times: int32 first, last, cells, tokens, first and last
// token of the rows, tiles of the key range: from, to, and the marked one.
// stdout: for each the marked tile's place, how many pairs follow, and the pairs
// (first key, key past the last) that are gone through.
#include <algorithm>
#include <type_traits>

#include "block.h"

#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_perm(a, b, pick) 0u
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, ...) c
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, ...) c
#define KV_TYPE_F32 0
#define KV_TYPE_F16 1
#define KV_TYPE_Q8_0 8
#define KV_TYPE_BF16 30
#include "odd_tiles.inc"

int main() {
    int h[9];
    while (fread(h, sizeof h, 1, stdin) == 1) {
        AttnArgs a{};
        a.first = h[0], a.last = h[1];
        Sequence q{};
        q.held = h[2], q.n_new = h[3], q.base = h[2] - h[3];
        const KeyTiles<true, 32> keys(a, q, h[4], h[5], (q.base + h[5] + 1 + 31) / 32);
        const int lo = h[6], hi = std::min(h[7], keys.n), t = lo + h[8] % (hi - lo);
        OddTiles odd(lo, hi);
        odd.add(t);
        std::vector<int> out = {keys.tile(t), 0};
        odd.each(keys, q.held, [&](int key, int end) {
            out.push_back(key);
            out.push_back(end);
        });
        out[1] = (out.size() - 2) / 2;
        give(out);
    }
    return 0;
}
