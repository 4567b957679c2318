// Paged KV cache on MI355X (include/kvc-cache.h): page bookkeeping on the
// device, and the copies of rows it asks for.
//
// Bookkeeping (extend, fork, free, the first step of compact) is one block of
// 16 waves: requests are a lane each for the checks and a wave each for their
// pages. It is latency bound; what it saves is the host round trip that would
// keep a serving step out of a captured graph. A page is free when its count
// is 0, so there is no free list to keep in step: an allocation scans the
// counts from page 0 until it has enough, which makes page numbers a function
// of the cache alone, and a call that needs no page does not scan.
//
// Rows move as bytes and are bound by HBM.
//
// Accepting the drafts of 16 sequences (cut, extend, write, compact: six
// launches) takes 49 us, most of it launches and these blocks' chains of loads;
// forking and extending samples, with the copy of their last pages, 112 us (96
// at a large copy's rate).
#include "kvc_codec.h"
#include "kvc_launch.h"

#include <stdint.h>

#include <initializer_list>

namespace kvc {

namespace {

constexpr int kPlan = 1024;               // threads of a bookkeeping block
constexpr int kWaves = kPlan / 64;
constexpr int kShared = 1 << 30;          // saved table entry: the page has other holders
constexpr int kMaxPages = 1 << 20;
constexpr int kMaxRows = 1 << 24;          // of a write or read: row numbers and a launch's threads stay in range

// Arrays and shapes of a cache as kernels take them.
struct Pages {
    int n_layers, n_pages, shift, max_seqs, max_pages, H;
    long long krow, vrow;   // bytes
    char * K;
    char * V;
    float * bias;
    int * table;
    int * len;
    int * refs;
};

// One request's move, written by the plan kernels into the workspace.
struct Job {
    int seq;
    int first;     // first cell written
    int start;     // cells before it keep their place (they move only with a replaced page)
    int kept;      // cells that move up behind start
    int k0;        // their first index
    int end;       // cells before the call
    int apart;     // 1: no page is both read and written, so rows may move in any order
};

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// Sum of v over the block's threads before this one; *total the whole sum.
__device__ int block_scan(int v, int * lds, int * total) {
    const int lane = lane_id(), w = threadIdx.x >> 6;
    int x = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) lds[w] = x;
    __syncthreads();
    if (threadIdx.x < kWaves) {
        int y = lds[threadIdx.x];
        for (int o = 1; o < kWaves; o <<= 1) {
            const int z = __shfl_up(y, o);
            if ((int)threadIdx.x >= o) y += z;
        }
        lds[threadIdx.x] = y;
    }
    __syncthreads();
    const int before = (w ? lds[w - 1] : 0) + x - v;
    *total = lds[kWaves - 1];
    __syncthreads();
    return before;
}

// The lowest `want` free pages into list; returns how many there are of them.
__device__ int find_free(const Pages & c, int want, int * list, int * lds) {
    int found = 0;
    for (int p0 = 0; p0 < c.n_pages && found < want; p0 += 4 * kPlan) {
        const int p = p0 + 4 * (int)threadIdx.x;
        int free[4], n = 0;
        for (int j = 0; j < 4; j++) {
            free[j] = p + j < c.n_pages && c.refs[p + j] == 0;
            n += free[j];
        }
        int total;
        int at = found + block_scan(n, lds, &total);
        for (int j = 0; j < 4; j++) {
            if (free[j]) {
                if (at < want) list[at] = p + j;
                at++;
            }
        }
        found += total;
    }
    __syncthreads();
    return found < want ? found : want;
}

// Grants pages in request order, all of a request's or none. need < 0: a bad
// request. Returns the first place in the free list, or -1 (not granted);
// *missing is the number of pages that were not there.
__device__ int grant(const Pages & c, int n, int need, int * list, int * lds, int * slots, int * missing) {
    const int i = threadIdx.x;
    int total;
    const int mine = need > 0 ? need : 0;
    int at = block_scan(mine, lds, &total);
    *missing = 0;
    if (total == 0) return need < 0 ? -1 : 0;
    const int have = find_free(c, total, list, lds);
    if (have < total) {   // (rare) one thread goes through the requests
        slots[i] = i < n ? mine : 0;
        __syncthreads();
        if (i == 0) {
            int used = 0;
            for (int j = 0; j < n; j++) {
                const int k = slots[j];
                if (used + k <= have) {
                    slots[j] = used;
                    used += k;
                } else {
                    slots[j] = -(k - (have - used));
                }
            }
        }
        __syncthreads();
        at = slots[i];
        if (at < 0) {
            *missing = -at;
            at = -1;
        }
        __syncthreads();
    }
    return need < 0 ? -1 : at;
}

// The pages of all requests as one list: first[r] is where request r's count[r]
// pages begin (in `first`), *total their number. A bookkeeping call is a chain
// of loads, and a thread per page makes it one chain for all requests.
__device__ const int * page_pairs(const int * count, int * first, int * lds, int * total) {
    const int i = threadIdx.x;
    const int at = block_scan(count[i], lds, total);
    first[i] = at;
    __syncthreads();
    return first;
}
// the request of entry x: the last one that begins at or before it
__device__ int request_of(const int * first, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// seqs[i], or -1 when out of range or named by an earlier request
__device__ int request_seq(const Pages & c, int n, const int * seqs, int * ids) {
    const int i = threadIdx.x;
    int s = -1;
    if (i < n) {
        s = seqs[i];
        if (s < 0 || s >= c.max_seqs) s = -1;
    }
    ids[i] = s;
    __syncthreads();
    if (s >= 0)
        for (int j = 0; j < i; j++)
            if (ids[j] == s) {
                s = -1;
                break;
            }
    __syncthreads();
    return s;
}

__device__ __forceinline__ bool good_page(const Pages & c, int p) { return p >= 0 && p < c.n_pages; }

__global__ __launch_bounds__(256) void k_cache_reset(Pages c) {
    const long long step = (long long)gridDim.x * blockDim.x, t0 = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    for (long long i = t0; i < (long long)c.max_seqs * c.max_pages; i += step) c.table[i] = -1;
    for (long long i = t0; i < c.max_seqs; i += step) c.len[i] = 0;
    for (long long i = t0; i < c.n_pages; i += step) c.refs[i] = 0;
}

// Reserves cells. A request's new pages are table columns have-copied .. of
// its sequence, where copied is 1 when the last page is partly filled and
// shared; that page's cells become a move job (identity, the old page in
// saved[job][0]). granted (or nullptr) names the sequences whose request is
// done, for the calls behind this one.
__global__ __launch_bounds__(kPlan) void k_cache_extend(Pages c, int n, const int * seqs, const int * count,
                                                        int * status, int * granted, Job * jobs, int * saved, int * list) {
    __shared__ int lds[kWaves], ids[kPlan], slots[kPlan], r_col[kPlan], r_need[kPlan], r_at[kPlan];
    const int i = threadIdx.x;
    const int page = 1 << c.shift;
    const int seq = request_seq(c, n, seqs, ids);
    const long long room = (long long)c.max_pages << c.shift;
    int need = -1, old = 0, add = 0, copied = 0, last = -1;
    if (seq >= 0) {
        old = c.len[seq];
        add = count[i];
        if (old >= 0 && old <= room && add >= 0 && old + (long long)add <= room) {
            const int have = (int)(((long long)old + page - 1) >> c.shift);
            const int want = (int)(((long long)old + add + page - 1) >> c.shift);
            need = want - have;
            if ((old & (page - 1)) && add > 0) {
                last = c.table[(long long)seq * c.max_pages + have - 1];
                if (!good_page(c, last)) {
                    need = -1;
                } else if (c.refs[last] > 1) {
                    copied = 1;
                    need++;
                }
            }
        }
    }
    __syncthreads();
    int missing;
    const int at = grant(c, n, need, list, lds, slots, &missing);
    const bool done = need >= 0 && at >= 0;
    r_need[i] = done ? need : 0;
    r_at[i] = at;
    r_col[i] = (int)(((long long)old + page - 1) >> c.shift) - copied;
    ids[i] = seq;
    if (i < n) {
        status[i] = done ? 0 : (missing ? missing : KVC_REQ_BAD);
        if (granted) granted[i] = done ? seq : -1;
        Job j{};
        if (done && copied) {
            j = Job{seq, old & ~(page - 1), old, 0, 0, old, 1};
            saved[(long long)i * c.max_pages] = last;
            atomicSub(&c.refs[last], 1);
        }
        jobs[i] = j;
        if (done && add) c.len[seq] = old + add;
    }
    __syncthreads();
    int total;
    const int * first = page_pairs(r_need, slots, lds, &total);
    for (int x = i; x < total; x += kPlan) {
        const int r = request_of(first, n, x), j = x - first[r];
        const int p = list[r_at[r] + j];
        c.table[(long long)ids[r] * c.max_pages + r_col[r] + j] = p;
        c.refs[p] = 1;
    }
}

__global__ __launch_bounds__(kPlan) void k_cache_fork(Pages c, int n, const int * src, const int * dst, int * status) {
    __shared__ int lds[kWaves], ids[kPlan], from[kPlan], held[kPlan], at[kPlan];
    const int i = threadIdx.x;
    const int to = request_seq(c, n, dst, ids);
    int a = -1, cells = 0;
    if (to >= 0) {
        a = src[i];
        cells = a >= 0 && a < c.max_seqs ? c.len[a] : -1;
        if (a == to || cells < 0 || cells > ((long long)c.max_pages << c.shift) || c.len[to] != 0) a = -1;
    }
    from[i] = a;
    held[i] = a >= 0 ? (int)(((long long)cells + (1 << c.shift) - 1) >> c.shift) : 0;
    ids[i] = to;
    __syncthreads();
    if (i < n) status[i] = a >= 0 ? 0 : KVC_REQ_BAD;
    if (a >= 0) c.len[to] = cells;
    // (a source that this call fills was empty before it: no page of it is read)
    int total;
    const int * first = page_pairs(held, at, lds, &total);
    for (int x = i; x < total; x += kPlan) {
        const int r = request_of(first, n, x), j = x - first[r];
        const int p = c.table[(long long)from[r] * c.max_pages + j];
        c.table[(long long)ids[r] * c.max_pages + j] = p;
        if (good_page(c, p)) atomicAdd(&c.refs[p], 1);
    }
}

__global__ __launch_bounds__(kPlan) void k_cache_free(Pages c, int n, const int * seqs) {
    __shared__ int lds[kWaves], ids[kPlan], held[kPlan], at[kPlan];
    const int i = threadIdx.x;
    const int seq = request_seq(c, n, seqs, ids);
    const int cells = seq >= 0 ? c.len[seq] : 0;
    ids[i] = seq;
    const long long pages = cells <= 0 ? 0 : ((long long)cells + (1 << c.shift) - 1) >> c.shift;
    held[i] = pages < c.max_pages ? (int)pages : c.max_pages;
    __syncthreads();
    if (seq >= 0) c.len[seq] = 0;
    int total;
    const int * first = page_pairs(held, at, lds, &total);
    for (int x = i; x < total; x += kPlan) {
        const int r = request_of(first, n, x);
        int * t = c.table + (long long)ids[r] * c.max_pages + (x - first[r]);
        const int p = *t;
        *t = -1;
        if (good_page(c, p)) atomicSub(&c.refs[p], 1);
    }
}

// Compaction, first step: which pages a request writes, fresh ones for those
// that have other holders, the pages behind its new end given back, and its
// move job. saved[r] holds the table before the call from column start/page
// on, with kShared set where the page is replaced.
__global__ __launch_bounds__(kPlan) void k_cache_plan_compact(Pages c, int n, const int * seqs, const int * start,
                                                              const int * cu, int n_idx, int * status,
                                                              Job * jobs, int * saved, int * list) {
    __shared__ int lds[kWaves], ids[kPlan], slots[kPlan], r_first[kPlan], r_written[kPlan], r_held[kPlan],
        r_need[kPlan];
    const int i = threadIdx.x;
    const int page = 1 << c.shift;
    const int seq = request_seq(c, n, seqs, ids);
    int from = 0, kept = 0, old = 0, k0 = 0;
    bool good = false;
    if (seq >= 0) {
        old = c.len[seq];
        from = start[i];
        k0 = cu[i];
        const long long k = (long long)cu[i + 1] - k0;
        good = old >= 0 && old <= ((long long)c.max_pages << c.shift) && from >= 0 && from <= old && k0 >= 0 && k >= 0 &&
               k <= old - from && cu[i + 1] <= n_idx;
        kept = good ? (int)k : 0;
    }
    const int first = from >> c.shift;
    const int held = good ? (int)(((long long)old + page - 1) >> c.shift) : 0;
    const int end = (int)(((long long)from + kept + page - 1) >> c.shift);   // pages after the call
    ids[i] = good ? seq : -1;
    r_first[i] = first;
    r_written[i] = kept > 0 ? end : first;   // columns first .. written-1 are written
    r_held[i] = held;
    __syncthreads();
    for (int r = i >> 6; r < n; r += kWaves) {
        if (ids[r] < 0) continue;
        const int * t = c.table + (long long)ids[r] * c.max_pages;
        int shared = 0, bad = 0;
        for (int j = r_first[r] + lane_id(); j < r_held[r]; j += 64) {
            const int p = t[j];
            const bool ok = good_page(c, p);
            const bool other = ok && j < r_written[r] && c.refs[p] > 1;
            saved[(long long)r * c.max_pages + j - r_first[r]] = ok ? (other ? p | kShared : p) : -1;
            shared += other;
            bad |= !ok;
        }
        for (int o = 32; o; o >>= 1) {
            shared += __shfl_xor(shared, o);
            bad |= __shfl_xor(bad, o);
        }
        if (lane_id() == 0) r_need[r] = bad ? -1 : shared;
    }
    __syncthreads();
    const int need = i < n && ids[i] >= 0 ? r_need[i] : -1;
    int missing;
    const int at = grant(c, n, need, list, lds, slots, &missing);
    const bool done = need >= 0 && at >= 0;
    if (i < n) status[i] = done ? 0 : (missing ? missing : KVC_REQ_BAD);
    __syncthreads();
    slots[i] = done ? at : -1;
    if (i < n) {
        Job j{};
        if (done) {
            // the cells before start on a page that is replaced move with it
            const bool lead = kept > 0 && (from & (page - 1)) && (saved[(long long)i * c.max_pages] & kShared);
            j = Job{seq, lead ? from & ~(page - 1) : from, from, kept, k0, old, need == r_written[i] - first};
            c.len[seq] = from + kept;
        }
        jobs[i] = j;
    }
    // (every count that decides a page was read before the barrier above)
    __syncthreads();
    for (int r = i >> 6; r < n; r += kWaves) {
        if (ids[r] < 0 || slots[r] < 0) continue;
        int * t = c.table + (long long)ids[r] * c.max_pages;
        const int first_r = r_first[r], written = r_written[r], lane = lane_id();
        // columns that stay: all before `keep`
        const int keep = jobs[r].kept > 0 ? written : (jobs[r].start + page - 1) >> c.shift;
        int next = slots[r];
        for (int j0 = first_r; j0 < r_held[r]; j0 += 64) {
            const int j = j0 + lane;
            const int p = j < r_held[r] ? saved[(long long)r * c.max_pages + j - first_r] : 0;
            const bool fresh = j < r_held[r] && (p & kShared);
            const unsigned long long m = __ballot(fresh);
            if (fresh) {
                const int q = list[next + __popcll(m & ((1ull << lane) - 1))];
                t[j] = q;
                c.refs[q] = 1;
                atomicSub(&c.refs[p & ~kShared], 1);
            } else if (j < r_held[r] && j >= keep) {
                t[j] = -1;
                atomicSub(&c.refs[p], 1);
            }
            next += __popcll(m);
        }
    }
}

// What a move kernel takes besides the jobs.
struct Move {
    const int * idx;
    long long ld_idx;
    const char * v;              // V rows given by the caller, or nullptr
    long long v_layer, v_row, v_head;
    int v_head_bytes;
    const float * beta;
    long long b_layer, b_head;
};

constexpr int kCells = 1024;   // cells whose places a block works out at a time
constexpr int kBatch = 16;     // rows a thread loads before it stores them

// Places of cells c0 .. c0+kCells-1 of a job (all threads; barriers inside).
// A place is a row of the pool, page * page_size + cell, or -1: left out (an
// index that does not fit leaves out all of its cell, given values too).
// from_caller: the kept cells' sources are rows of the caller's array, and
// rows of the pool stand as -2 - place.
__device__ void cell_places(const Pages & c, const Job & j, const int * saved, const int * idx, bool from_caller,
                            int c0, int hi, int * src, int * dst) {
    const int mask = (1 << c.shift) - 1, lead = j.start - j.first, col0 = j.start >> c.shift;
    const int * t = c.table + (long long)j.seq * c.max_pages;
    __syncthreads();
    for (int e = threadIdx.x; e < kCells; e += blockDim.x) {
        const int k = c0 + e;
        int a = -1, b = -1;
        if (k < hi) {
            const int to = j.first + k;
            const int q = t[to >> c.shift];
            if (good_page(c, q)) b = (q << c.shift) + (to & mask);
            const bool kept = k >= lead;
            int from = to;
            if (kept) {
                // (an index below its place would read a row that is already overwritten)
                const int x = idx[j.k0 + k - lead];
                from = x >= k - lead && x < j.end - j.start ? j.start + x : -1;
            }
            if (kept && from_caller) {
                if (from >= 0) a = k - lead;
            } else {
                const int p = from >= 0 ? saved[(from >> c.shift) - col0] : -1;
                if (p >= 0) a = ((p & ~kShared) << c.shift) + (from & mask);
                if (a == b) a = -1;
                if (a >= 0 && from_caller) a = -2 - a;
            }
            if (b < 0) a = -1;
        }
        src[e] = a;
        dst[e] = b;
    }
    __syncthreads();
}

// Moves the rows of the jobs: K, V and bias, all layers. A thread owns columns
// of sizeof(U) bytes and takes the cells in ascending order, kBatch loads
// ahead of their stores. A kept cell never moves down, so a row is read before
// it is overwritten without a barrier between threads; jobs that read and
// write different pages are cut into gridDim.x / col_blocks cell ranges too.
// Bound by HBM (a fifth of 32768 cells of 32 layers kept on fresh pages, with
// given V and bias: 389 us, 4.4 TB/s; 411 with the plan and the fork before it),
// or by the latency of one column's chain where a long job moves in place: the
// same cells of a sequence that shares no page take 1.7 ms.
template <class U>
__global__ __launch_bounds__(256) void k_cache_move(Pages c, const Job * jobs, const int * saved,
                                                    Move mv, int col_blocks) {
    __shared__ int src[kCells], dst[kCells];
    const int job = blockIdx.z;
    const Job j = jobs[job];
    const int m = j.start - j.first + j.kept;
    if (m <= 0) return;
    const int layer = blockIdx.y % c.n_layers, what = blockIdx.y / c.n_layers;   // what: 0 K, 1 V, 2 bias
    const int cb = blockIdx.x % col_blocks, part = blockIdx.x / col_blocks;
    const bool from_caller = what == 1 ? mv.v != nullptr : what == 2 && mv.beta;
    const int parts = j.apart || from_caller ? gridDim.x / col_blocks : 1;
    const int per = ((m + parts - 1) / parts + 63) & ~63;
    const long long lo64 = (long long)part * per;
    if (lo64 >= m) return;
    const int lo = (int)lo64, hi = m - lo < per ? m : lo + per;
    const int * idx = mv.idx + layer * mv.ld_idx;
    saved += (long long)job * c.max_pages;
    if (what == 2) {
        const long long pool = ((long long)layer * c.n_pages << c.shift) * c.H;
        const int mask = (1 << c.shift) - 1;
        for (int c0 = lo; c0 < hi; c0 += kCells) {
            cell_places(c, j, saved, idx, from_caller, c0, hi, src, dst);
            for (int h = cb; h < c.H; h += col_blocks) {
                float x[kCells / 256];
                for (int e = 0; e < kCells / 256; e++) {
                    const int a = src[e * 256 + threadIdx.x];
                    const int row = from_caller ? -2 - a : a;
                    if (from_caller && a >= 0)
                        x[e] = mv.beta[layer * mv.b_layer + h * mv.b_head + j.k0 + a];
                    else if (a != -1)
                        x[e] = c.bias[pool + (((long long)(row >> c.shift) * c.H + h) << c.shift) + (row & mask)];
                }
                // a cell that one thread overwrites another may still have to read
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
                for (int e = 0; e < kCells / 256; e++) {
                    const int b = dst[e * 256 + threadIdx.x];
                    if (src[e * 256 + threadIdx.x] != -1)
                        c.bias[pool + (((long long)(b >> c.shift) * c.H + h) << c.shift) + (b & mask)] = x[e];
                }
            }
        }
        return;
    }
    const long long row_bytes = what ? c.vrow : c.krow;
    char * pool = (what ? c.V : c.K) + ((long long)layer * c.n_pages << c.shift) * row_bytes;
    const long long col = ((long long)cb * 256 + threadIdx.x) * (int)sizeof(U);
    const bool mine = col < row_bytes;
    const char * given = nullptr;
    if (from_caller)
        given = mv.v + layer * mv.v_layer + (long long)j.k0 * mv.v_row + (col / mv.v_head_bytes) * mv.v_head +
                col % mv.v_head_bytes;
    for (int c0 = lo; c0 < hi; c0 += kCells) {
        cell_places(c, j, saved, idx, from_caller, c0, hi, src, dst);
        if (!mine) continue;
        const int n = hi - c0 < kCells ? hi - c0 : kCells;
        U x[kBatch], y[kBatch];
        auto load = [&](U * v, int e0) {
#pragma unroll
            for (int e = 0; e < kBatch; e++) {
                const int a = e0 + e < n ? src[e0 + e] : -1;
                if (a == -1) continue;
                v[e] = *reinterpret_cast<const U *>(!from_caller ? pool + a * row_bytes + col
                                                    : a >= 0     ? given + a * mv.v_row
                                                                 : pool + (-2 - a) * row_bytes + col);
            }
        };
        load(x, 0);
        for (int e0 = 0; e0 < n; e0 += kBatch) {
            load(y, e0 + kBatch);
#pragma unroll
            for (int e = 0; e < kBatch; e++)
                if (e0 + e < n && src[e0 + e] != -1) *reinterpret_cast<U *>(pool + dst[e0 + e] * row_bytes + col) = x[e];
#pragma unroll
            for (int e = 0; e < kBatch; e++) x[e] = y[e];
        }
    }
}

// Row r of the call's packed rows: its sequence's cell, as a row of the pool
// (page * page_size + cell), or -1. All threads; the answer for the block's
// rows r0 .. r0+rows-1 (kRows at most) in place[]. The threads look for the
// rows' sequences; then a thread a row follows its chain of loads. A page of
// more than one sequence takes no rows: a reservation that was granted never
// ends in one, so these would be cells that were there before.
constexpr int kRows = 8;
__device__ void new_row_places(const Pages & c, int n, const int * seqs, const int * cu, int r0, int rows, int n_rows, int * place) {
    if (threadIdx.x < kRows) place[threadIdx.x] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int a = cu[i], b = cu[i + 1];
        const int lo = a > r0 ? a : r0;
        int hi = b < r0 + rows ? b : r0 + rows;
        if (hi > n_rows) hi = n_rows;
        for (int r = lo; r < hi; r++) place[r - r0] = i;
    }
    __syncthreads();
    if (threadIdx.x < kRows) {
        const int i = place[threadIdx.x], s = i >= 0 ? seqs[i] : -1;
        int at = -1;
        if (s >= 0 && s < c.max_seqs) {
            const int held = c.len[s];
            const long long cell = (long long)held - cu[i + 1] + r0 + threadIdx.x;
            if (cell >= 0 && cell < held && held <= (long long)c.max_pages << c.shift) {
                const int p = c.table[(long long)s * c.max_pages + (cell >> c.shift)];
                if (good_page(c, p) && c.refs[p] <= 1) at = (p << c.shift) + (int)(cell & ((1 << c.shift) - 1));
            }
        }
        place[threadIdx.x] = at;
    }
    __syncthreads();
}

struct RowSource {
    const char * data;
    long long ld_layer, ld_row;
};

// New rows of the cache's own type: blocks of `rows` rows of one layer. A copy:
// bound by HBM, or by the launch where the rows are few.
template <class U>
__global__ __launch_bounds__(256) void k_cache_write(Pages c, int layer0, int n, const int * seqs, const int * cu,
                                                     int n_rows, int rows, RowSource k, RowSource v) {
    __shared__ int place[kRows];
    const int r0 = blockIdx.x * rows, layer = layer0 + blockIdx.y;
    new_row_places(c, n, seqs, cu, r0, rows, n_rows, place);
    const int kc = (int)(c.krow / (int)sizeof(U)), vc = (int)(c.vrow / (int)sizeof(U));
    const long long base = (long long)layer * c.n_pages << c.shift;
#pragma unroll 4
    for (unsigned w = threadIdx.x; w < (unsigned)rows * (unsigned)(kc + vc); w += 256) {
        const int e = (int)(w / (unsigned)(kc + vc)), x = (int)(w % (unsigned)(kc + vc));
        if (place[e] < 0) continue;
        const bool is_v = x >= kc;
        const RowSource & s = is_v ? v : k;
        const int col = is_v ? x - kc : x;
        const U val = *reinterpret_cast<const U *>(s.data + blockIdx.y * s.ld_layer + (long long)(r0 + e) * s.ld_row +
                                                   (long long)col * (int)sizeof(U));
        char * to = is_v ? c.V + (base + place[e]) * c.vrow : c.K + (base + place[e]) * c.krow;
        *reinterpret_cast<U *>(to + (long long)col * (int)sizeof(U)) = val;
    }
    if (c.bias)
        for (int w = threadIdx.x; w < rows * c.H; w += 256) {
            const int p = place[w / c.H], h = w % c.H;
            if (p >= 0)
                c.bias[((((long long)layer * c.n_pages + (p >> c.shift)) * c.H + h) << c.shift) +
                       (p & ((1 << c.shift) - 1))] = 0.0f;
        }
}

// F32, F16 or BF16 value i of a row
__device__ __forceinline__ float row_value(const char * row, int type, long long i) {
    if (type == KV_TYPE_F32) return reinterpret_cast<const float *>(row)[i];
    const unsigned short u = reinterpret_cast<const unsigned short *>(row)[i];
    if (type == KV_TYPE_BF16) return __uint_as_float((unsigned)u << 16);
    return (float)__builtin_bit_cast(_Float16, u);
}

// New rows encoded into Q8_0 (kv_quantize_row's arithmetic): four lanes a
// block of 32, eight values each. 4096 F16 rows of 32 layers (8 x 128): 104 us;
// 16 rows of one layer 16 us (two blocks, eight rounds of their threads).
__global__ __launch_bounds__(256) void k_cache_write_q8(Pages c, int layer0, int n, const int * seqs, const int * cu,
                                                        int n_rows, int type, RowSource k, RowSource v) {
    __shared__ int place[kRows];
    const int r0 = blockIdx.x * kRows, layer = layer0 + blockIdx.y;
    new_row_places(c, n, seqs, cu, r0, kRows, n_rows, place);
    const int kb = (int)(c.krow / 34), vb = (int)(c.vrow / 34);
    const long long base = (long long)layer * c.n_pages << c.shift;
    const int work = kRows * (kb + vb) * 4;
    // (whole waves take part in the shuffles; lanes past the end write nothing)
    for (int w0 = 0; w0 < work; w0 += 256) {
        const int w = w0 + (int)threadIdx.x, q = w & 3;
        const int e = w < work ? w / 4 / (kb + vb) : 0, x = w / 4 % (kb + vb);
        const bool on = w < work && place[e] >= 0, is_v = x >= kb;
        const int blk = is_v ? x - kb : x;
        float val[8], amax = 0.0f;
        const RowSource & s = is_v ? v : k;
        const char * row = s.data + blockIdx.y * s.ld_layer + (long long)(r0 + e) * s.ld_row;
        for (int i = 0; i < 8; i++) {
            val[i] = on ? row_value(row, type, blk * 32 + q * 8 + i) : 0.0f;
            const float t = fabsf(val[i]);
            if (t > amax) amax = t;
        }
        const float o1 = __shfl_xor(amax, 1);
        amax = o1 > amax ? o1 : amax;
        const float o2 = __shfl_xor(amax, 2);
        amax = o2 > amax ? o2 : amax;
        if (!on) continue;
        const float d = amax / 127.0f;
        const float id = d != 0.0f ? 127.0f / amax : 0.0f;
        uint16_t * o = reinterpret_cast<uint16_t *>((is_v ? c.V + (base + place[e]) * c.vrow
                                                          : c.K + (base + place[e]) * c.krow) + blk * 34);
        if (q == 0) o[0] = f32_to_f16_ref(d);
        for (int i = 0; i < 4; i++) {
            const uint8_t a = (uint8_t)(int8_t)roundf(fmax_std(-128.0f, fmin_std(127.0f, val[2 * i] * id)));
            const uint8_t b = (uint8_t)(int8_t)roundf(fmax_std(-128.0f, fmin_std(127.0f, val[2 * i + 1] * id)));
            o[1 + 4 * q + i] = (uint16_t)(a | (uint16_t)b << 8);
        }
    }
    if (c.bias)
        for (int w = threadIdx.x; w < kRows * c.H; w += 256) {
            const int p = place[w / c.H], h = w % c.H;
            if (p >= 0)
                c.bias[((((long long)layer * c.n_pages + (p >> c.shift)) * c.H + h) << c.shift) +
                       (p & ((1 << c.shift) - 1))] = 0.0f;
        }
}

// Cells start .. start+count-1 of one sequence as contiguous rows. A copy: 32768
// cells of 32 layers (bf16, 8 x 128) in 1.68 ms, 5.2 TB/s.
template <class U>
__global__ __launch_bounds__(256) void k_cache_read(Pages c, int seq, int start, int count, char * K, char * V,
                                                    float * bias) {
    __shared__ int place[kRows];
    const int k0 = blockIdx.x * kRows, layer = blockIdx.y;
    if (threadIdx.x < kRows) {
        const long long cell = (long long)start + k0 + threadIdx.x;
        const int held = c.len[seq];
        int p = -1;
        if (cell < held && cell < (long long)c.max_pages << c.shift) {
            const int q = c.table[(long long)seq * c.max_pages + (cell >> c.shift)];
            if (good_page(c, q)) p = (q << c.shift) + (int)(cell & ((1 << c.shift) - 1));
        }
        place[threadIdx.x] = p;
    }
    __syncthreads();
    const int rows = count - k0 < kRows ? count - k0 : kRows;
    const int kc = K ? (int)(c.krow / (int)sizeof(U)) : 0, vc = V ? (int)(c.vrow / (int)sizeof(U)) : 0;
    const long long base = (long long)layer * c.n_pages << c.shift, out = (long long)layer * count + k0;
    for (long long w = threadIdx.x; w < (long long)rows * (kc + vc); w += 256) {
        const int e = (int)(w / (kc + vc)), x = (int)(w % (kc + vc));
        const bool is_v = x >= kc;
        const long long col = (long long)(is_v ? x - kc : x) * (int)sizeof(U), row = is_v ? c.vrow : c.krow;
        U val{};
        if (place[e] >= 0) val = *reinterpret_cast<const U *>((is_v ? c.V : c.K) + (base + place[e]) * row + col);
        *reinterpret_cast<U *>((is_v ? V : K) + (out + e) * row + col) = val;
    }
    if (bias)
        for (int w = threadIdx.x; w < kRows * c.H; w += 256) {
            const int e = w % kRows, h = w / kRows, p = place[e];
            if (e >= rows) continue;
            bias[((long long)layer * c.H + h) * count + k0 + e] =
                p < 0 ? 0.0f
                      : c.bias[((((long long)layer * c.n_pages + (p >> c.shift)) * c.H + h) << c.shift) +
                               (p & ((1 << c.shift) - 1))];
        }
}

bool paged_type(int t) { return t == KV_TYPE_F32 || t == KV_TYPE_F16 || t == KV_TYPE_BF16 || t == KV_TYPE_Q8_0; }

int shift_of(int page_size) {
    for (int s = 4; s <= 10; s++)
        if (page_size == 1 << s) return s;
    return -1;
}

Pages pages_of(const kvc_cache * c) {
    Pages p{};
    p.n_layers = c->n_layers; p.n_pages = c->n_pages; p.shift = shift_of(c->page_size);
    p.max_seqs = c->max_seqs; p.max_pages = c->max_pages; p.H = c->n_head_kv;
    p.krow = (long long)kv_quant_row_bytes(c->k_type, c->n_head_kv * c->d_k);
    p.vrow = (long long)kv_quant_row_bytes(c->v_type, c->n_head_kv * c->d_v);
    p.K = static_cast<char *>(c->K); p.V = static_cast<char *>(c->V); p.bias = c->bias;
    p.table = c->table; p.len = c->len; p.refs = c->refs;
    return p;
}

// Workspace of extend and compact: the jobs, each request's table before the
// call, the free pages found.
struct PlanWork {
    Job * jobs;
    int * saved;
    int * list;
    size_t bytes;
};
PlanWork plan_work(const kvc_cache * c, int n, void * ws) {
    PlanWork w{};
    char * p = static_cast<char *>(ws);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char * q = p ? p + off : nullptr;
        off += (bytes + 255) & ~(size_t)255;
        return q;
    };
    w.jobs = reinterpret_cast<Job *>(take(sizeof(Job) * n));
    w.saved = reinterpret_cast<int *>(take(sizeof(int) * (size_t)n * c->max_pages));
    w.list = reinterpret_cast<int *>(take(sizeof(int) * (size_t)c->n_pages));
    w.bytes = off;
    return w;
}

int check_requests(int n) {
    if (n < 0) return -2;
    return n > KVC_CACHE_MAX_REQUESTS ? KV_COMPACT_E_UNSUPPORTED : 0;
}

// Widest unit of 16, 4 or 2 bytes that divides every one of the values
int unit_of(std::initializer_list<long long> v) {
    long long m = 0;
    for (long long x : v) m |= x;
    return m % 16 == 0 ? 16 : m % 4 == 0 ? 4 : 2;
}

typedef unsigned U16 __attribute__((ext_vector_type(4)));

// The rows of the jobs that a plan kernel wrote, at most `cells` of each.
bool launch_move(const kvc_cache * c, const Pages & p, const PlanWork & w, int n, long long cells, const Move & mv,
                 int unit, hipStream_t st) {
    const long long row = p.krow > p.vrow ? p.krow : p.vrow;
    const int col_blocks = (int)((row / unit + 255) / 256);
    const int kinds = p.bias ? 3 : 2;
    // cell ranges of jobs that may be cut: at least 64 cells each, and no
    // more than fill the GPU (16 blocks a CU)
    const long long blocks = (long long)col_blocks * c->n_layers * kinds * n;
    long long parts = (cells + 63) / 64, most = (4096 + blocks - 1) / blocks;
    parts = parts < most ? parts : most;
    const dim3 grid((unsigned)(col_blocks * (parts > 1 ? parts : 1)), (unsigned)(c->n_layers * kinds), (unsigned)n);
    if (unit == 16)
        return launch(k_cache_move<U16>, grid, dim3(256), st, p, (const Job *)w.jobs,
                      (const int *)w.saved, mv, col_blocks);
    if (unit == 4)
        return launch(k_cache_move<unsigned>, grid, dim3(256), st, p, (const Job *)w.jobs,
                      (const int *)w.saved, mv, col_blocks);
    return launch(k_cache_move<unsigned short>, grid, dim3(256), st, p, (const Job *)w.jobs,
                  (const int *)w.saved, mv, col_blocks);
}

}  // namespace

int check_cache(const kvc_cache * c) {
    if (!c || !c->K || !c->V || !c->table || !c->len || !c->refs) return -1;
    if (c->n_layers <= 0 || c->n_pages <= 0 || c->max_seqs <= 0 || c->max_pages <= 0 || c->n_head_kv <= 0 ||
        c->d_k <= 0 || c->d_v <= 0)
        return -2;
    if (shift_of(c->page_size) < 0 || c->n_pages > kMaxPages || c->max_pages > kMaxPages || c->d_k > 256 ||
        c->d_v > 256 || c->n_head_kv > 65535 || c->n_layers > 16384 || !paged_type(c->k_type) ||
        !paged_type(c->v_type))
        return KV_COMPACT_E_UNSUPPORTED;
    if ((c->k_type == KV_TYPE_Q8_0 && c->d_k % 32) || (c->v_type == KV_TYPE_Q8_0 && c->d_v % 32))
        return KV_COMPACT_E_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(c->K) | reinterpret_cast<uintptr_t>(c->V) | reinterpret_cast<uintptr_t>(c->bias)) & 15)
        return KV_COMPACT_E_UNSUPPORTED;
    return 0;
}

}  // namespace kvc

using namespace kvc;

extern "C" {

int kvc_cache_reset(const kvc_cache * c, void * stream) {
    if (int rc = check_cache(c)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    return launch(k_cache_reset, dim3(256), dim3(256), st, pages_of(c)) ? 0 : KV_COMPACT_E_DEVICE;
}

size_t kvc_cache_workspace(const kvc_cache * c, int n) {
    if (check_cache(c) || n <= 0 || n > KVC_CACHE_MAX_REQUESTS) return 0;
    return plan_work(c, n, nullptr).bytes;
}

int kvc_cache_extend_granted(const kvc_cache * c, int n, const int * seqs, const int * count, int * status,
                             int * granted, void * ws, size_t ws_bytes, void * stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_requests(n)) return rc;
    if (n == 0) return 0;
    if (!seqs || !count || !status || !ws) return -1;
    const PlanWork w = plan_work(c, n, ws);
    if (w.bytes > ws_bytes) return KVC_E_SCRATCH;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    const Pages p = pages_of(c);
    // (whole pages are 16-byte aligned, rows of a page may not be)
    if (!launch(k_cache_extend, dim3(1), dim3(kPlan), st, p, n, seqs, count, status, granted, w.jobs, w.saved,
                w.list) ||
        !launch_move(c, p, w, n, c->page_size, Move{}, unit_of({p.krow, p.vrow}), st))
        return KV_COMPACT_E_DEVICE;
    return 0;
}

int kvc_cache_extend(const kvc_cache * c, int n, const int * seqs, const int * count, int * status, void * ws,
                     size_t ws_bytes, void * stream) {
    return kvc_cache_extend_granted(c, n, seqs, count, status, nullptr, ws, ws_bytes, stream);
}

int kvc_cache_write(const kvc_cache * c, int layer, int n_layers, int n, const int * seqs, const int * cu, int n_rows,
                    int src_type, const kvc_rows * K, const kvc_rows * V, void * stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_requests(n)) return rc;
    if (layer < 0 || n_layers < 0 || n_rows < 0 || layer > c->n_layers - n_layers) return -2;
    if (n_rows > kMaxRows) return KV_COMPACT_E_UNSUPPORTED;
    if (n == 0 || n_layers == 0 || n_rows == 0) return 0;
    if (!seqs || !cu || !K || !V || !K->data || !V->data) return -1;
    const bool encode = src_type != KV_TYPE_Q8_0 && c->k_type == KV_TYPE_Q8_0 && c->v_type == KV_TYPE_Q8_0 &&
                        paged_type(src_type);
    if (!encode && (src_type != c->k_type || src_type != c->v_type)) return KV_COMPACT_E_UNSUPPORTED;
    const long long any = reinterpret_cast<long long>(K->data) | K->ld_layer | K->ld_row |
                          reinterpret_cast<long long>(V->data) | V->ld_layer | V->ld_row;
    if (any & (src_type == KV_TYPE_F32 ? 3 : 1)) return KV_COMPACT_E_UNSUPPORTED;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    const Pages p = pages_of(c);
    const RowSource k{static_cast<const char *>(K->data), K->ld_layer, K->ld_row};
    const RowSource v{static_cast<const char *>(V->data), V->ld_layer, V->ld_row};
    const dim3 grid((unsigned)((n_rows + kRows - 1) / kRows), (unsigned)n_layers);
    bool ok;
    if (encode) {
        ok = launch(k_cache_write_q8, grid, dim3(256), st, p, layer, n, seqs, cu, n_rows, src_type, k, v);
    } else {
        const int unit = unit_of({any, p.krow, p.vrow});
        // eight rows a block find their cells together; two where that would leave CUs idle
        // (F16, 8 x 128; blocks of two and of eight, us: 16 to 2048 rows of a layer 4.0 and
        // 5.8, 8192 rows 6.1 both, 16384 rows 8.8 and 7.0; 32 layers of 60 rows 5.4 and 7.4,
        // of 158 rows 11.4 both, of 383 rows 23.6 and 22.6)
        const int rows = (long long)((n_rows + kRows - 1) / kRows) * n_layers < 1024 ? 2 : kRows;
        const dim3 grid((unsigned)((n_rows + rows - 1) / rows), (unsigned)n_layers);
        ok = unit == 16  ? launch(k_cache_write<U16>, grid, dim3(256), st, p, layer, n, seqs, cu, n_rows, rows, k, v)
             : unit == 4 ? launch(k_cache_write<unsigned>, grid, dim3(256), st, p, layer, n, seqs, cu, n_rows, rows, k, v)
                         : launch(k_cache_write<unsigned short>, grid, dim3(256), st, p, layer, n, seqs, cu, n_rows, rows, k, v);
    }
    return ok ? 0 : KV_COMPACT_E_DEVICE;
}

int kvc_cache_fork(const kvc_cache * c, int n, const int * src, const int * dst, int * status, void * stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_requests(n)) return rc;
    if (n == 0) return 0;
    if (!src || !dst || !status) return -1;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    return launch(k_cache_fork, dim3(1), dim3(kPlan), st, pages_of(c), n, src, dst, status) ? 0 : KV_COMPACT_E_DEVICE;
}

int kvc_cache_free(const kvc_cache * c, int n, const int * seqs, void * stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_requests(n)) return rc;
    if (n == 0) return 0;
    if (!seqs) return -1;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    return launch(k_cache_free, dim3(1), dim3(kPlan), st, pages_of(c), n, seqs) ? 0 : KV_COMPACT_E_DEVICE;
}

int kvc_cache_compact(const kvc_cache * c, int n, const int * seqs, const int * start, const int * cu, int n_idx,
                      const int * idx, long long ld_idx, const kvc_values * v, const kvc_betas * beta, int * status,
                      void * ws, size_t ws_bytes, void * stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_requests(n)) return rc;
    if (n_idx < 0 || ld_idx < 0) return -2;
    if (n == 0) return 0;
    if (!seqs || !start || !cu || !status || !ws || (n_idx && !idx) || (v && !v->data) || (beta && !beta->data))
        return -1;
    if (beta && !c->bias) return KV_COMPACT_E_UNSUPPORTED;
    const PlanWork w = plan_work(c, n, ws);
    if (w.bytes > ws_bytes) return KVC_E_SCRATCH;
    const Pages p = pages_of(c);
    Move mv{idx, ld_idx};
    long long any = p.krow | p.vrow;
    if (v) {
        mv.v = static_cast<const char *>(v->data);
        mv.v_layer = v->ld_layer; mv.v_row = v->ld_row; mv.v_head = v->ld_head;
        mv.v_head_bytes = (int)(p.vrow / c->n_head_kv);
        const long long given = reinterpret_cast<long long>(v->data) | v->ld_layer | v->ld_row | v->ld_head;
        if (given & (c->v_type == KV_TYPE_F32 ? 3 : 1)) return KV_COMPACT_E_UNSUPPORTED;
        any |= given | mv.v_head_bytes;
    }
    if (beta) {
        mv.beta = beta->data; mv.b_layer = beta->ld_layer; mv.b_head = beta->ld_head;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    if (!launch(k_cache_plan_compact, dim3(1), dim3(kPlan), st, p, n, seqs, start, cu, n_idx, status, w.jobs,
                w.saved, w.list))
        return KV_COMPACT_E_DEVICE;
    if (n_idx && !launch_move(c, p, w, n, n_idx, mv, unit_of({any}), st)) return KV_COMPACT_E_DEVICE;
    return 0;
}

int kvc_cache_read(const kvc_cache * c, int seq, int start, int count, void * K_out, void * V_out, float * bias_out,
                   void * stream) {
    if (int rc = check_cache(c)) return rc;
    if (seq < 0 || seq >= c->max_seqs || start < 0 || count < 0) return -2;
    if (count > kMaxRows || (bias_out && !c->bias)) return KV_COMPACT_E_UNSUPPORTED;
    if (count == 0 || (!K_out && !V_out && !bias_out)) return 0;
    if ((reinterpret_cast<uintptr_t>(K_out) | reinterpret_cast<uintptr_t>(V_out)) & 1) return KV_COMPACT_E_UNSUPPORTED;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice dev(st);
    if (!dev.ok) return KV_COMPACT_E_DEVICE;
    const Pages p = pages_of(c);
    const long long any = reinterpret_cast<long long>(K_out) | reinterpret_cast<long long>(V_out) | p.krow | p.vrow;
    char * k = static_cast<char *>(K_out);
    char * o = static_cast<char *>(V_out);
    const dim3 grid((unsigned)((count + kRows - 1) / kRows), (unsigned)c->n_layers);
    const int unit = unit_of({any});
    const bool ok = unit == 16  ? launch(k_cache_read<U16>, grid, dim3(256), st, p, seq, start, count, k, o, bias_out)
                    : unit == 4 ? launch(k_cache_read<unsigned>, grid, dim3(256), st, p, seq, start, count, k, o, bias_out)
                                : launch(k_cache_read<unsigned short>, grid, dim3(256), st, p, seq, start, count, k, o,
                                         bias_out);
    return ok ? 0 : KV_COMPACT_E_DEVICE;
}

}  // extern "C"
