/*
 * dsv4_speculative.h - what a speculative decoding step needs next to the decode
 * attention of dsv4_attn.h: attention of a tree of drafted tokens, sampling, and the
 * pages of the cache around them.  No counterpart in the reference project.
 *
 * The conventions are those of dsv4_attn.h: raw device pointers of the caller, nothing
 * allocated, work enqueued on `stream`, 0 or a cudaError_t value returned, an optional
 * `status` array of DSV4_STATUS_WORDS int32.
 */
#ifndef DSV4_SPECULATIVE_H_
#define DSV4_SPECULATIVE_H_

#include "dsv4_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Tree decode.  The T drafted nodes of request b attend, in one softmax each, to every entry
 * [0, kv_len[b]) of the request (through the block table) and to those of the first
 * win_len[b] rows of its window buffer that the node's mask names: bit w % 32 of word w / 32 of
 * tree_mask[b][t] is set where node t sees window row w.  The window buffer holds the last
 * committed tokens and the drafted ones; a node's bits leave out tokens that have slid out
 * of its window and drafts that are not its ancestors.  A node that sees nothing gives 0 and
 * an lse of -inf.  Arithmetic, preconditions and NaN rows as for dsv4_hca_dense_decode_fwd: |q| < 65504, block scales <= 146 (below 6e-5, FP16's smallest normal
 * number, they lose accuracy), no e4m3 NaN in a row that any node sees.
 *
 * num_splits >= 1: a static grid of that many pieces per row group (> 1 needs partial_o and partial_lse of
 * num_splits * B * T * H rows, as dsv4_attn_workspace_bytes(B, T * H, ...) says).  num_splits = 0: `sched` is a plan;
 * with make_plan it is made by this call first, else it was made by dsv4_attn_plan (kind HCA, this B, s_q = 1, H = T * H,
 * these lengths).  sched, partial_o and partial_lse then have the sizes dsv4_attn_sched_bytes(B, T * H, 0, 0, ...)
 * reports.
 */
typedef struct Dsv4HcaTreeDecodeParams {
    int32_t B;
    int32_t T;                  /* nodes per request (1: a plain decode step) */
    int32_t H;                  /* query heads */
    int32_t max_pages;
    int32_t win_cap;            /* rows per request in win_pool */
    int32_t mask_words;         /* 32-bit words per node of tree_mask; window rows beyond them are seen by no node */
    int32_t num_splits;
    float   sm_scale;
    int32_t make_plan;
    int32_t reserved0;
    int64_t num_pages;
    const void*    q;           /* bf16  [B, T, H, 576] */
    const void*    kv_pool;     /* uint8 [num_pages, 64, 656] */
    const int32_t* block_table; /* int32 [B, max_pages] */
    const int32_t* kv_len;      /* int32 [B] */
    const void*    win_pool;    /* uint8 [B, win_cap, 656] */
    const int32_t* win_len;     /* int32 [B] */
    const int32_t* tree_mask;   /* int32 [B, T, mask_words] */
    const float*   attn_sink;   /* optional float [H] */
    void*          out;         /* bf16  [B, T, H, 512] */
    float*         lse;         /* optional float [B, T, H] */
    float*         partial_o;
    float*         partial_lse;
    int32_t*       status;
    void*          sched;
    int64_t        sched_bytes; /* read with make_plan */
    void*          rows;        /* optional workspace of dsv4_hca_tree_rows_bytes(), 32-byte aligned: the entries are dequantised into it once, and all of a
                                   request's nodes read them there; without it every group of 128 (node, head) rows dequantises them for itself */
    int64_t        rows_bytes;
} Dsv4HcaTreeDecodeParams;

int64_t dsv4_hca_tree_rows_bytes(int B, int max_pages, int win_cap);

int dsv4_hca_tree_decode_fwd(const Dsv4HcaTreeDecodeParams* p, void* stream);

/*
 * Pages of the cache.  A pool is [layers][num_pages][64][656] bytes (layers = 1: one layer's pool); one block table
 * and one count per page serve all layers.  refs[p] counts the block-table slots that hold page p; a page with a
 * count of 0 is free.  Numbers that a call names below are device arrays; a negative page, entry or request leaves
 * its item out, one that is out of range leaves it out and is reported (DSV4_STATUS_BAD_INDEX).
 */
#define DSV4_STATUS_NO_PAGE 10  /* a fork found no free page: the child has the full pages only (its length says so) */

typedef struct Dsv4KvPagesParams {
    void*          pool;        /* copy, fork, compact, move */
    int64_t        num_pages;
    int64_t        layers;      /* >= 1 */
    int64_t        entries;     /* move: entries per layer (the pool is then [layers][entries][656]: cache or window) */
    int32_t        B;           /* fork, free, compact: requests = rows of block_table */
    int32_t        max_pages;
    int32_t        n;           /* items of src / dst */
    int32_t        reserved0;
    const int32_t* src;         /* copy: pages; fork: parents; free: requests; move: entries */
    const int32_t* dst;         /* copy: pages; fork: children; move: entries */
    int32_t*       block_table; /* [B, max_pages] */
    int32_t*       kv_len;      /* [B] */
    int32_t*       refs;        /* [num_pages] */
    int32_t*       new_table;   /* compact: [B, max_pages], may be block_table */
    int32_t*       new_refs;    /* compact: [num_pages], may be refs */
    int32_t*       count;       /* compact: [1], live pages */
    int32_t*       scratch;     /* compact: 2 * num_pages + 1 */
    int32_t*       status;
} Dsv4KvPagesParams;

#define DSV4_STATUS_OVERLAP 11  /* lists of a copy or a move overlap where they must not */

/* Page src[i] to page dst[i] in every layer.  No page is named twice among dst, nor in both lists: the latter is reported (DSV4_STATUS_OVERLAP), and what
 * such pages hold afterwards is unspecified. */
int dsv4_kv_pages_copy(const Dsv4KvPagesParams* p, void* stream);

/* Child dst[i] becomes a copy of parent src[i]: it shares the parent's full pages (one reference more each), and
 * where the parent's last page is partly filled gets a page of its own with a copy of the entries in use: free pages
 * in ascending order, for the children in their order.  The child's table row and length are overwritten: whatever
 * pages it held must have been freed.  Children are distinct, and no child is a parent. */
int dsv4_kv_pages_fork(const Dsv4KvPagesParams* p, void* stream);

/* The pages of requests src[i] (distinct) are given back: one reference less each; table rows -1, lengths 0. */
int dsv4_kv_pages_free(const Dsv4KvPagesParams* p, void* stream);

/* Live pages move to the front of the pool: with `count` of them, the k-th live page from number `count` on goes to
 * the k-th free page below it, in every layer.  new_table and new_refs are the tables afterwards. */
int dsv4_kv_pages_compact(const Dsv4KvPagesParams* p, void* stream);

/* Entry src[i] to entry dst[i] in every layer, as if all of them were read before any is written: accepted drafts to their places, also where those
 * are other accepted drafts' (rows that close up, a window that slides).  No entry is named twice among dst.  Lists of more than 16,384 entries must not
 * overlap: if they do, nothing is moved, and it is reported (DSV4_STATUS_OVERLAP). */
int dsv4_kv_entries_move(const Dsv4KvPagesParams* p, void* stream);

/*
 * Sampling from logits [N, V] with given random numbers.  For row n with temperature t > 0, l_max its largest logit:
 *     e_i = exp((l_i - l_max) * (1 / t)),  w_i = floor(2^40 e_i)
 *   tokens are ordered by logit, then by index (the lower first);
 *   top_k > 0:       the first top_k of them are kept;
 *   top_p < 1:       of those, the ones before which less than max(1, floor(p * total weight kept so far)) lies;
 *   min_p > 0:       of those, the ones with e_i >= min(min_p, 1);
 * and the token is the first, in the order of the vocabulary, up to which more than floor(u * total weight kept) lies.
 * The weights are integers, so that sums do not depend on their order and a call gives the same token whatever the
 * batch around it; what they leave out is less than V * 2^-40 of the largest probability.  p and u enter as multiples
 * of 2^-24 (rounded down; u is clamped to [0, 1)).  t <= 0 or NaN: the largest logit, lowest index.  top_k <= 0, top_p >= 1
 * or NaN and min_p <= 0 or NaN leave their filter out; so do null pointers (temperature: 1).  A NaN logit counts as -inf;
 * a row of nothing but -inf gives token -1 and logprob -inf.  logprob is the logarithm of the probability the token was
 * drawn with, log(w / total weight kept), 0 for a greedy row.
 */
#define DSV4_DTYPE_F32  0
#define DSV4_DTYPE_BF16 1
#define DSV4_DTYPE_F16  2
typedef struct Dsv4SampleParams {
    int32_t N;
    int32_t V;                  /* at most 2^22 */
    int32_t dtype;              /* of the logits */
    int32_t reserved0;
    int64_t stride_n;           /* elements between rows, any value >= V */
    const void*    logits;
    const float*   u;           /* [N] */
    const float*   temperature; /* optional [N] */
    const int32_t* top_k;       /* optional [N] */
    const float*   top_p;       /* optional [N] */
    const float*   min_p;       /* optional [N] */
    int32_t*       token;       /* [N] */
    float*         logprob;     /* optional [N] */
} Dsv4SampleParams;

int dsv4_sample_fwd(const Dsv4SampleParams* p, void* stream);

#ifdef __cplusplus
}
#endif
#endif  /* DSV4_SPECULATIVE_H_ */
