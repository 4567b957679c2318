// The attention kernels in the forms with a window (include/kvc-cache.h, kvc_window).
#include "kvc_attn_kernels.h"

namespace kvc {

bool run_attn_window(const AttnArgs & a, int type, int qt, int whole, int rt, bool careful, long long blocks, hipStream_t st) {
    return run_attn<true>(a, type, qt, whole, rt, careful, blocks, st);
}

}  // namespace kvc
