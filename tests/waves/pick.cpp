// kvc_cache_pick's kernels (cut out of kvc_evict.hip by the test that builds
// this) on the CPU, lane by lane.
//
// stdin: int32 own (keys by a launch of their own), first wave to run, layers,
// sequences, H, room, n, n_idx, recent, most, groups, max_len; len, seqs, start,
// keep; weights. stdout: cu, granted, status, indices [groups][n_idx].
#include "block.h"

#define KVC_REQ_BAD (-2)
#include "pick.inc"

int main() {
    const std::vector<int> h = take<int>(12);
    PickArgs p{};
    const int own = h[0], first = h[1], seqs = h[3];
    p.n_layers = h[2], p.max_seqs = seqs, p.H = h[4], p.room = h[5], p.n = h[6], p.n_idx = h[7], p.recent = h[8];
    p.most = h[9], p.groups = h[10], p.max_len = h[11];
    const std::vector<int> len = take<int>(seqs), which = take<int>(p.n), start = take<int>(p.n), keep = take<int>(p.n);
    const std::vector<float> w = take<float>((size_t)p.n_layers * seqs * p.H * p.room);
    p.stride = (p.max_len + 3) / 4 * 4;
    std::vector<int> cu(p.n + 1, 99), granted(p.n, 99), status(p.n, 99), idx((size_t)p.groups * p.n_idx, -7);
    std::vector<u4> keys((size_t)p.groups * p.n * p.stride / 4);
    p.seqs = which.data(), p.start = start.data(), p.keep = keep.data(), p.len = len.data(), p.weight = w.data();
    p.idx = idx.data(), p.ld_idx = p.n_idx, p.cu = cu.data(), p.granted = granted.data(), p.status = status.data();
    p.keys = reinterpret_cast<unsigned *>(keys.data());
    p.parts = p.max_len / 1024 + 1;
    const unsigned units = p.groups * p.n;
    if (own)
        for (blockIdx.x = 0; blockIdx.x < units * p.parts; blockIdx.x++) run_block(4, 0, [&] { k_cell_keys(p); });
    for (blockIdx.x = 0; blockIdx.x < units; blockIdx.x++)
        run_block(kWaves, first, [&] { own ? k_pick<false>(p) : k_pick<true>(p); });
    give(cu);
    give(granted);
    give(status);
    give(idx);
    return 0;
}
