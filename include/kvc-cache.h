/*
 * Paged KV cache and attention on MI355X: the operators around a compaction.
 * Additive to the reference ABI (the reference leaves cache and attention to
 * llama.cpp; its compaction results, include/kv-compact-api.h:221-241, are
 * consumed there).
 *
 *   kvc_attn_prompt    causal attention over whole prompts (packed sequences)
 *   kvc_cache_*        pages: reserve, write, fork, free, compact, read
 *   kvc_attn_cache     attention of new or drafted tokens over the cache,
 *                      with the per-head bias (beta) a compaction fits
 *
 * A serving step: kvc_cache_extend reserves the new tokens' cells, each layer
 * writes its K and V rows (kvc_cache_write) and attends (kvc_attn_cache).
 * Compaction: kvc_cache_read gathers a sequence's rows for
 * kvc_compact_layers_device or kvc_compact_quantized_layers_device, and
 * kvc_cache_compact keeps the cells they select, with the refitted values
 * and beta.
 *
 * All pointers inside the structs are device (HBM) memory of the stream's
 * device. Every call queues its work on `stream` (NULL: the default stream of
 * the current device), returns without waiting, allocates nothing and may be
 * captured into a HIP graph. The calls keep no state of their own: two of
 * them may run at once when they share no output, workspace or cache that one
 * of them changes. The structs are read before the call returns.
 *
 * Return codes as in kv-compact-api.h: 0; -1 NULL argument; -2 bad dimension;
 * KV_COMPACT_E_UNSUPPORTED (-5) a type or size outside the limits below;
 * KV_COMPACT_E_DEVICE (-6) no usable GPU or a failed launch; KVC_E_SCRATCH
 * (-7) the workspace is too small. Nothing is launched on an error.
 */
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "kv-compact-api.h"
#include "kv-compact-device.h"   /* KVC_E_SCRATCH */

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the cache ------------------------------------------------------------
 * A cell is one token's K and V rows of all layers. Cells of a sequence stand
 * in pages of page_size cells; page p of every layer belongs to the same
 * sequences. The caller owns every array:
 *   K     [n_layers][n_pages][page_size][k_row bytes]  rows in codec k_type,
 *   V     [n_layers][n_pages][page_size][v_row bytes]  heads concatenated
 *   bias  [n_layers][n_pages][n_head_kv][page_size] float, or NULL: no bias
 *   table [max_seqs][max_pages]  page of each page_size cells, -1 past the end
 *   len   [max_seqs]             cells held
 *   refs  [n_pages]              sequences that hold the page; 0: free
 * k_row bytes is kv_quant_row_bytes(k_type, n_head_kv * d_k), likewise V.
 * Types: F32, F16, BF16, Q8_0 (its head width a multiple of 32). Where k_type
 * and v_type differ, kvc_cache_write and kvc_attn_cache return
 * KV_COMPACT_E_UNSUPPORTED: the caller fills such a cache and reads it by
 * kernels of its own, and these calls reserve, share, move and gather the rows.
 * page_size: a power of two from 16 to 1024. n_pages <= 2^20. d_k, d_v <= 256.
 * K, V and bias 16-byte aligned, the workspaces too (hipMalloc's are).
 * New pages are the lowest free ones, in request order, so that equal calls
 * on equal caches give equal tables. */
typedef struct kvc_cache {
    int n_layers, n_pages, page_size, max_seqs, max_pages;
    int n_head_kv, d_k, d_v, k_type, v_type;
    void *  K;
    void *  V;
    float * bias;
    int *   table;
    int *   len;
    int *   refs;
} kvc_cache;

/* All pages free, all sequences empty. */
int kvc_cache_reset(const kvc_cache * c, void * stream);

/* Requests of one call: at most KVC_CACHE_MAX_REQUESTS. status (device
 * int[n]): 0 done; > 0 that many pages were missing and nothing was done for
 * this request; KVC_REQ_BAD the sequence number, count or table size does not
 * fit, or an earlier request of the call names the same sequence. A request
 * is refused by itself: the others are done. */
#define KVC_CACHE_MAX_REQUESTS 1024
#define KVC_REQ_BAD (-2)

/* Bytes of device workspace for a call of n requests (extend, compact). */
size_t kvc_cache_workspace(const kvc_cache * c, int n);

/* Sequence seqs[i] grows by count[i] >= 0 cells, whose rows kvc_cache_write
 * fills. A last page that is partly filled and shared is copied first. */
int kvc_cache_extend(const kvc_cache * c, int n, const int * seqs, const int * count, int * status,
                     void * ws, size_t ws_bytes, void * stream);

/* The same, and granted (device int[n], NULL: not wanted) becomes seqs[i]
 * where the request was done and -1 where it was refused. A step whose calls
 * are queued behind the reservation without a look at its status gives
 * kvc_cache_write and kvc_attn_cache this array as their seqs: rows of a
 * refused request are then written nowhere, and its tokens see nothing. */
int kvc_cache_extend_granted(const kvc_cache * c, int n, const int * seqs, const int * count, int * status,
                             int * granted, void * ws, size_t ws_bytes, void * stream);

/* Rows of the last cells of each sequence, layers layer .. layer+n_layers-1.
 * Sequence seqs[i] takes rows cu[i] .. cu[i+1]-1 (cu: device int[n+1]) into
 * its last cu[i+1]-cu[i] cells, oldest first; n_rows = cu[n], known on the
 * host (rows at or past it are not written). The bias of written cells
 * becomes 0. K and V rows of src_type: a cache of the same type takes the
 * bytes, a Q8_0 cache also F32, F16 and BF16 rows, encoded as by
 * kv_quantize_row. Row r of layer layer+j at byte j*ld_layer + r*ld_row;
 * both strides multiples of 2 (F32: 4). n_rows <= 2^24. A sequence number
 * that the cache does not have takes no rows; each other is named once.
 * The cells are those that the last kvc_cache_extend reserved. Where it
 * refused, the last cells are older ones, so that sequence is not named here
 * (kvc_cache_extend_granted leaves it out). Pages that another sequence holds
 * too are not written: a sequence is forked before it is extended or after
 * its rows are written, not in between. */
typedef struct kvc_rows {
    const void * data;
    long long ld_layer, ld_row;   /* bytes */
} kvc_rows;
int kvc_cache_write(const kvc_cache * c, int layer, int n_layers, int n, const int * seqs, const int * cu,
                    int n_rows, int src_type, const kvc_rows * K, const kvc_rows * V, void * stream);

/* Sequence dst[i], empty, comes to hold the cells of src[i]: the pages are
 * shared. Requests see the cache as it was before the call. */
int kvc_cache_fork(const kvc_cache * c, int n, const int * src, const int * dst, int * status, void * stream);

/* Sequence seqs[i] becomes empty; pages that no other holds are free. An
 * empty sequence may be named, a sequence named twice is freed once. */
int kvc_cache_free(const kvc_cache * c, int n, const int * seqs, void * stream);

/* Compaction: of sequence seqs[i], the cells before start[i] stay, and of the
 * others those at start[i] + idx[k], k = cu[i] .. cu[i+1]-1, move up behind
 * them; what follows is dropped (no indices: the sequence is cut to start[i]).
 * Layer l's indices are idx + l*ld_idx (ld_idx 0: the same cells in every
 * layer), ascending within a sequence, each at least k - cu[i] and inside the
 * sequence (where one is not, its cell's K, V and bias keep what their place
 * on the page held, also with v and beta). n_idx = cu[n], known on the host: a
 * request whose cu[i+1] is past it is refused (KVC_REQ_BAD), as is one that
 * asks for more cells than the sequence has behind start[i].
 * v (NULL: the kept cells' own rows) gives the V rows: head h of row k of
 * layer l at byte l*ld_layer + k*ld_row + h*ld_head, in the cache's V type;
 * address and strides multiples of 2 (F32: 4).
 * beta (NULL: the kept cells' own bias) gives the bias:
 * beta[l*ld_layer + h*ld_head + k]. The outputs of
 * kvc_compact_layers_device (C_v: ld_row 4*d_v, ld_head 4*t*d_v, ld_layer
 * 4*H*t*d_v; beta: ld_head t, ld_layer H*t) and of the quantized entry fit as
 * they are. Rows move within the sequence's pages; a page that is shared is
 * replaced by a free one. start[i] is the same in every layer. v and beta
 * overlap no array of the cache. */
typedef struct kvc_values {
    const void * data;
    long long ld_layer, ld_row, ld_head;   /* bytes */
} kvc_values;
typedef struct kvc_betas {
    const float * data;
    long long ld_layer, ld_head;           /* floats */
} kvc_betas;
int kvc_cache_compact(const kvc_cache * c, int n, const int * seqs, const int * start, const int * cu,
                      int n_idx, const int * idx, long long ld_idx, const kvc_values * v,
                      const kvc_betas * beta, int * status, void * ws, size_t ws_bytes, void * stream);

/* Cells start .. start+count-1 of sequence seq, all layers, as contiguous
 * rows: K_out [n_layers][count][k_row bytes], V_out likewise, bias_out
 * [n_layers][n_head_kv][count] (any may be NULL). Cells past the sequence's
 * end read as zero bytes. count <= 2^24. */
int kvc_cache_read(const kvc_cache * c, int seq, int start, int count, void * K_out, void * V_out,
                   float * bias_out, void * stream);

/* ---- attention ------------------------------------------------------------
 * Token i, head h of an array: data + i*ld_tok + h*ld_head elements, the d
 * values of a head side by side. Any strides (of K and V tokens: from 0 to
 * under 2^24 bytes, a cache's rows too) and base alignment; rows that
 * are 16-byte aligned (base and strides) with d_k and d_v multiples of 8 are
 * the fast ones. n_head is a multiple of n_head_kv: query heads h*g ..
 * h*g+g-1 read KV head h. d_k, d_v from 1 to 256. Sums and softmax statistics
 * are fp32; F16 and BF16 round the softmax weights to that type before the
 * product with V (a Q8_0 cache: to fp16), and the result once. Over a Q8_0
 * cache scores take the blocks' codes exactly and their scales in fp32; BF16
 * queries lose the bits of elements under 2^-28 of their row's largest; values
 * of V are scale times code rounded to fp16 where the result is BF16. A call has at
 * most 2^30 rows (n_tok * n_head), and a launch's blocks limit it: prompts to
 *   n_head_kv * (ceil(n_tok * n_head / n_head_kv / R) + n_seq) < 2^23,
 * R = 128 for F16 and BF16 whose q, k, v and o are all in aligned rows, else 32
 * where q, k and v are and heads are up to 128 wide, else 16; a cache call to
 *   n_head_kv * n_seq < 2^23.
 * o and lse overlap no input. A row that sees no cell gives zeros and lse
 * -inf. lse = log(sum exp(scale q.k + bias)), float [n_tok][n_head], may be
 * NULL. scale 0: 1/sqrt(d_k). */
typedef struct kvc_heads {
    void *    data;
    long long ld_tok, ld_head;   /* elements */
} kvc_heads;

/* Causal self-attention of packed prompts. Sequence s is tokens cu[s] ..
 * cu[s+1]-1 (cu: device int[n_seq+1], ascending); token i sees the tokens of
 * its sequence up to itself. Tokens outside every sequence are left as they
 * were in o and lse. type: F16, BF16 or F32, for q, k, v and o. */
typedef struct kvc_prompt_args {
    kvc_heads q, k, v, o;
    float *     lse;
    const int * cu;
    int type, n_seq, n_tok, n_head, n_head_kv, d_k, d_v;
    float scale;
} kvc_prompt_args;
int kvc_attn_prompt(const kvc_prompt_args * a, void * stream);

/* Attention over one layer of a cache. Sequence seqs[s] (NULL: s) has tokens
 * cu[s] .. cu[s+1]-1 (cu: device int[n_seq+1], ascending), whose rows are the last cells of the sequence: n_new =
 * cu[s+1]-cu[s] of len. Every token sees the cells before those. Of the last
 * n_new, token i sees cell j when bit j % 64 of mask[i_row*mask_words + j/64]
 * is set (a tree of drafts: a token's ancestors and itself), without a mask
 * when j <= i. Cells past mask_words*64 are not seen. A sequence with more
 * tokens than cells sees nothing, and so does a token of a bad sequence
 * number or the part of a sequence on a bad page number. Tokens outside every
 * sequence are left as they were.
 * type: F32 with an F32 cache, F16 with F16, BF16 with BF16, F16 or BF16 with
 * Q8_0 (k_type and v_type alike). max_new and max_len are what the launch is
 * shaped for: the most tokens and cells of a sequence (larger ones are right,
 * and slower). */
typedef struct kvc_cache_attn_args {
    kvc_heads q, o;
    float *     lse;
    const int * seqs;
    const int * cu;
    const uint64_t * mask;
    int mask_words;
    int layer, type, n_seq, n_tok, n_head, max_new, max_len;
    float scale;
} kvc_cache_attn_args;
size_t kvc_attn_cache_workspace(const kvc_cache * c, const kvc_cache_attn_args * a);
int kvc_attn_cache(const kvc_cache * c, const kvc_cache_attn_args * a, void * ws, size_t ws_bytes, void * stream);

#ifdef __cplusplus
}
#endif
