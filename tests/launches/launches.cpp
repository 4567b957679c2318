// What the cache's calls hand to their launches, with a runtime that records
// instead of launching: addresses far into large caches, and launches of any size
// that arguments can announce. (The undefined-behaviour sanitizer sees the entry
// points' sums and products; the kernels are not built.)
#include "../../kv-compact_amd/csrc/kvc_attn_kernels.h"

#include <cstdio>
#include <cstring>
#include <vector>

namespace {

int launches = 0, failures = 0;
char argument[1024];   // the last launch's, as much of it as is asked for
size_t wanted = 0;
long long threads_most = 0;

#define CHECK(c)                                                            \
    do {                                                                    \
        if (!(c)) {                                                         \
            fprintf(stderr, "check failed: %s (line %d)\n", #c, __LINE__);  \
            failures++;                                                     \
        }                                                                   \
    } while (0)

char * const base = reinterpret_cast<char *>(1ull << 20);   // (never looked into)
template <class T> T * at(unsigned long long byte) { return reinterpret_cast<T *>(base + byte); }

kvc_cache cache(int layers, int seqs, int H, int pages, int page, int type) {
    kvc_cache c{};
    c.n_layers = layers, c.n_pages = 1 << 10, c.page_size = page, c.max_seqs = seqs, c.max_pages = pages;
    c.n_head_kv = H, c.d_k = c.d_v = 64, c.k_type = c.v_type = type;
    c.K = c.V = base, c.table = at<int>(0), c.len = at<int>(0), c.refs = at<int>(0);
    return c;
}
kvc_cache_attn_args attn(int layer, int type, int n_seq, int n_tok, int n_head, int max_new, int max_len) {
    kvc_cache_attn_args a{};
    a.q = kvc_heads{base, 64LL * n_head, 64}, a.o = a.q;
    a.lse = at<float>(0), a.cu = at<int>(0), a.layer = layer, a.type = type, a.n_seq = n_seq, a.n_tok = n_tok, a.n_head = n_head;
    a.max_new = max_new, a.max_len = max_len;
    return a;
}

}  // namespace

extern "C" {
hipError_t hipGetDevice(int * d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t * d) { *d = 0; return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipLaunchKernel(const void *, dim3 grid, dim3 block, void ** args, size_t, hipStream_t) {
    launches++;
    CHECK(grid.x > 0 && grid.y == 1 && grid.z == 1 && block.x % 64 == 0);
    const long long threads = (long long)grid.x * block.x;
    CHECK(threads < 1LL << 32);
    threads_most = threads > threads_most ? threads : threads_most;
    memcpy(argument, args[0], wanted);
    return hipSuccess;
}
size_t kv_quant_row_bytes(int type, int n) { return type == KV_TYPE_F32 ? 4ul * n : type == KV_TYPE_Q8_0 ? n / 32 * 34 : 2 * n; }
void ** __hipRegisterFatBinary(const void *) { return nullptr; }
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, void *, void *, int *) {}
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void **) {}
hipError_t __hipPopCallConfiguration(dim3 *, dim3 *, size_t *, hipStream_t *) { return hipSuccess; }
}

int main() {
    using namespace kvc;
    // weights of a late layer of many sequences: the launch's argument begins with the attention's, its weights come next
    wanted = sizeof(AttnArgs) + sizeof(float *);
    for (int layer : {0, 1, 2999, 16383}) {
        const kvc_cache c = cache(16384, 1 << 20, 2, 3, 16, KV_TYPE_F16);
        const kvc_cache_attn_args a = attn(layer, KV_TYPE_F16, 2, 2, 4, 1, 48);
        const kvc_weigh_args w = {at<float>(0), 1.0f, 0, 0};
        CHECK(kvc_cache_weigh(&c, &a, nullptr, &w, nullptr) == 0);
        float * to;
        memcpy(&to, argument + sizeof(AttnArgs), sizeof to);
        CHECK(to == at<float>(4ull * layer * (1 << 20) * 2 * 48));
    }
    wanted = 0;
    // a list for each layer of one sequence: one launch; one for all layers: the keys by blocks of their own, too
    for (int layers : {1, 8, 32}) {
        const kvc_cache c = cache(layers, 4, 8, 128, 64, KV_TYPE_F16);
        kvc_pick_args k{};
        k.seqs = k.start = k.keep = at<int>(0), k.weight = at<float>(0), k.idx = k.cu = k.granted = k.status = at<int>(0);
        k.n_idx = 1000, k.max_len = 5120;
        int before = launches;
        CHECK(kvc_cache_pick(&c, 1, &k, base, kvc_cache_pick_workspace(&c, 1, &k), nullptr) == 0);
        CHECK(launches - before == (layers > 1 ? 2 : 1));
        k.ld_idx = 1000;
        before = launches;
        CHECK(kvc_cache_pick(&c, 1, &k, base, kvc_cache_pick_workspace(&c, 1, &k), nullptr) == 0);
        CHECK(launches - before == 1);
    }
    // sizes that arguments can announce
    unsigned long long x = 88172645463325252ull;
    auto any = [&](long long most) {   // spread over the logarithm
        x ^= x << 13, x ^= x >> 7, x ^= x << 17;
        const int bits = x % 64;
        x ^= x << 13, x ^= x >> 7, x ^= x << 17;
        const long long v = (long long)(x >> 1 >> bits);
        return v > most || v < 0 ? most : v;
    };
    const int types[] = {KV_TYPE_F32, KV_TYPE_F16, KV_TYPE_BF16, KV_TYPE_Q8_0};
    for (int i = 0; i < 200000; i++) {
        const int type = types[any(1 << 20) % 4], H = 1 + (int)any(100) % 65, G = 1 + (int)any(64), n_seq = (int)any(1 << 23);
        kvc_cache c = cache(1 + (int)any(16383), 1 + (int)any((1u << 31) - 2), H, 1 + (int)any((1 << 20) - 1), 16 << any(6), type);
        while (4.0 * c.n_layers * c.max_seqs * H * c.max_pages * c.page_size > 0x1p46) c.max_seqs -= c.max_seqs / 2, c.max_pages -= c.max_pages / 2;
        kvc_cache_attn_args a = attn((int)any(c.n_layers - 1), type == KV_TYPE_Q8_0 ? KV_TYPE_F16 : type, n_seq, (int)any((1 << 30) / (H * G)), H * G,
                                     (int)any((1 << 30) / G), (int)any((1u << 31) - 1));
        if (i % 3 == 0) a.mask = at<uint64_t>(0), a.mask_words = (int)any((1u << 31) - 1);
        if (i % 5 == 0) a.q.ld_tok += 1;   // rows that are not aligned
        const kvc_window w = {(int)any((1u << 31) - 1), 1 + (int)any((1u << 31) - 2)};
        const kvc_weigh_args y = {at<float>(0), i % 2 ? 1.0f : 0.0f, (int)any((1u << 31) - 1), (int)any((1u << 31) - 1)};
        int rc = kvc_cache_weigh(&c, &a, i % 4 ? &w : nullptr, &y, nullptr);
        CHECK(rc == 0 || rc == KV_COMPACT_E_UNSUPPORTED);
        const size_t need = kvc_attn_cache_window_workspace(&c, &a, &w);
        rc = kvc_attn_cache_window(&c, &a, &w, base, need, nullptr);
        CHECK(rc == 0 || rc == KV_COMPACT_E_UNSUPPORTED);
        rc = kvc_attn_cache(&c, &a, base, kvc_attn_cache_workspace(&c, &a), nullptr);
        CHECK(rc == 0 || rc == KV_COMPACT_E_UNSUPPORTED);
        kvc_prompt_args p{};
        p.q = p.k = p.v = p.o = a.q, p.cu = at<int>(0), p.type = a.type, p.n_seq = n_seq, p.n_tok = a.n_tok, p.n_head = H * G;
        p.n_head_kv = H, p.d_k = p.d_v = 64;
        rc = kvc_attn_prompt_window(&p, &w, nullptr);
        CHECK(rc == 0 || rc == KV_COMPACT_E_UNSUPPORTED);
        const int n = 1 + (int)any(KVC_CACHE_MAX_REQUESTS - 1);
        kvc_pick_args k{};
        k.seqs = k.start = k.keep = at<int>(0), k.weight = at<float>(0), k.idx = k.cu = k.granted = k.status = at<int>(0);
        k.n_idx = (int)any((1u << 31) - 1), k.ld_idx = i % 2 ? k.n_idx + any(1ll << 40) : 0, k.recent = (int)any((1u << 31) - 1);
        k.max_len = (int)any((1u << 31) - 1);
        rc = kvc_cache_pick(&c, n, &k, base, kvc_cache_pick_workspace(&c, n, &k), nullptr);
        CHECK(rc == 0 || rc == KV_COMPACT_E_UNSUPPORTED);
        rc = kvc_cache_take_weights(&c, n, k.seqs, k.seqs, k.start, k.cu, k.n_idx, k.idx, k.ld_idx, nullptr, at<float>(0), nullptr);
        CHECK(rc == 0);
    }
    if (failures) {
        fprintf(stderr, "%d checks failed\n", failures);
        return 1;
    }
    printf("%d launches, up to %lld threads\n", launches, threads_most);
    return 0;
}
