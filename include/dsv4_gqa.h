/*
 * dsv4_gqa.h - attention over pages of ordinary K and V heads (grouped queries), next to the latent cache of dsv4_attn.h: what a
 * draft model, or a layer that does not compress, needs in a decoding step.  No counterpart in the reference project.
 *
 * The conventions are those of dsv4_attn.h: raw device pointers of the caller, nothing allocated, work enqueued on `stream`, 0 or a
 * cudaError_t value returned, an optional `status` array of DSV4_STATUS_WORDS int32.
 *
 * Pools.  K and V of one layer are [num_pages][64][Hkv][D] each, in BF16, FP16 or e4m3 (then value = e4m3 * scale[head], for any finite scale).  A block table
 * int32 [B][max_pages] maps a request's pages to pool pages; entry j of request b lies in page block_table[b][j / 64] at j % 64.  The page tables and
 * counts are those of dsv4_speculative.h: dsv4_kv_pages_free works on them as they are.  A page outside the pool, an entry outside the table: left out, not read, and
 * reported (DSV4_STATUS_BAD_INDEX).
 */
#ifndef DSV4_GQA_H_
#define DSV4_GQA_H_

#include "dsv4_attn.h"
#include "dsv4_speculative.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DSV4_DTYPE_E4M3 3

/*
 * Attention of new tokens.  kv_len[b] entries of request b exist, the last of them the new tokens' own (inserted before).  With T tokens each, token t of request b
 * stands at place p = kv_len[b] - T + t; packed (q_start given), the tokens of request b are rows q_start[b] .. q_start[b + 1] - 1 of q, and its last
 * token stands at kv_len[b] - 1.  Query head n reads KV head n / G.  A token sees the entries j <= p, with window > 0 only those with p - j < window or
 * j < first.  out = softmax(sm_scale q.k [, sink]) v; the sink, a logit per head, adds to the denominator.  A token that sees nothing gives 0 and an lse of -inf (natural
 * logarithm, without the sink).  Entries that no token of the request sees may hold anything; those that some token of the call sees must be finite.
 * Softmax weights are rounded to the type of V before they are multiplied (over e4m3 pages to FP16; in the prompts' kernel, which sizes choose, to q's type), all else is FP32.
 * Rows of q outside q_start[0] .. q_start[B] are left as they are in out and lse; offsets outside [0, rows] or that fall are clamped and reported.
 *
 * weights (tokens not packed): float [B][weight_stride], weight_stride >= max_pages * 64: to entry j of request b is added what it got from the call's tokens and heads,
 * the sum of their softmax weights (with the sink in the denominator).
 */
typedef struct Dsv4GqaParams {
    int32_t B;
    int32_t T;                  /* tokens per request (not packed) */
    int32_t Hkv;
    int32_t G;                  /* query heads per KV head */
    int32_t D;                  /* 64, 128 or 256 */
    int32_t max_pages;
    int32_t window;             /* 0: all entries */
    int32_t first;
    int32_t q_dtype;            /* DSV4_DTYPE_BF16 or _F16: q and out */
    int32_t kv_dtype;           /* the same, or DSV4_DTYPE_E4M3 */
    float   sm_scale;           /* > 0 */
    int32_t max_len;            /* optional: no kv_len is larger (steers the launch and the workspace; with weights, entries beyond it get none; packed tokens over e4m3 pages may
                                   not see entries beyond it, which are reported) */
    int64_t rows;               /* rows of q: B * T, or packed */
    int64_t num_pages;
    int64_t q_stride_b;         /* elements, multiples of 8 */
    int64_t q_stride_t;
    int64_t q_stride_h;
    const void*    q;           /* [B, T, Hkv * G, D] or [rows, Hkv * G, D], by its strides; D contiguous */
    const int32_t* q_start;     /* optional int32 [B + 1] */
    const void*    k_pool;
    const void*    v_pool;
    const int32_t* block_table;
    const int32_t* kv_len;      /* int32 [B] */
    const float*   k_scale;     /* e4m3: float [Hkv] */
    const float*   v_scale;
    const float*   attn_sink;   /* optional float [Hkv * G] */
    void*          out;         /* [rows, Hkv * G, D] */
    float*         lse;         /* optional float [rows, Hkv * G] */
    float*         weights;     /* optional */
    int64_t        weight_stride;
    void*          workspace;   /* dsv4_gqa_workspace_bytes(), 128-byte aligned */
    int64_t        workspace_bytes;
    int32_t*       status;
} Dsv4GqaParams;

/*
 * Follows from the sizes, kv_dtype, window, first, max_len, q's strides (whether they are 0: heads, tokens or requests that share their rows take other kernels), q_start and weights being
 * given, and the number of SMs; of pointers nothing else is looked at. -1: not such sizes.
 */
int64_t dsv4_gqa_workspace_bytes(const Dsv4GqaParams* p);

/* T tokens per request, q_start null: a decoding step, and the verification of a few drafted tokens. */
int dsv4_gqa_decode_fwd(const Dsv4GqaParams* p, void* stream);

/*
 * Packed tokens, q_start given: prompts, or pieces of them behind what is cached.  Of e4m3 pages a prompt's kernel has 16-bit copies in the workspace, which has room for B * max_pages * 64
 * entries, or B * max_len, up to 4 GiB: beyond that the call takes some requests at a time.
 */
int dsv4_gqa_prefill_fwd(const Dsv4GqaParams* p, void* stream);

/*
 * New rows of K and V, BF16 or FP16, into the pages: row t of request b becomes entry insert_pos[b] + t; rows as [B][T] (of which n_rows[b] are taken where that
 * is given) or packed by q_start.  Into e4m3 pools a value is divided by its head's scale and rounded to the nearest e4m3 (beyond 448: 448; 0 / 0: 0).
 * A place outside the table or the pool is left out and reported (code 16).
 */
typedef struct Dsv4GqaInsertParams {
    int32_t B;
    int32_t T;
    int32_t Hkv;
    int32_t D;                  /* a multiple of 8 */
    int32_t max_pages;
    int32_t src_dtype;          /* DSV4_DTYPE_BF16 or _F16 */
    int32_t kv_dtype;           /* the same, or DSV4_DTYPE_E4M3 */
    int32_t reserved0;
    int64_t rows;
    int64_t num_pages;
    int64_t k_stride_b;         /* elements, multiples of 8 */
    int64_t k_stride_t;
    int64_t k_stride_h;
    int64_t v_stride_b;
    int64_t v_stride_t;
    int64_t v_stride_h;
    const void*    k;
    const void*    v;
    const int32_t* q_start;     /* optional int32 [B + 1] */
    const int32_t* n_rows;      /* optional int32 [B] */
    void*          k_pool;
    void*          v_pool;
    const int32_t* block_table;
    const int32_t* insert_pos;  /* int32 [B] */
    const float*   k_scale;
    const float*   v_scale;
    int32_t*       status;
} Dsv4GqaInsertParams;

int dsv4_gqa_insert(const Dsv4GqaInsertParams* p, void* stream);

/*
 * Eviction by attention weight.  A request with more than keep entries (keep_each[b] where that is given) keeps its first `first` entries, its last `recent`, and of the others
 * those with the largest weights, keep in all (equal weights: the lower place; NaN counts as the least; if keep is less than first + recent, the first ones go before the
 * recent ones).  They close up in their order, in every layer of every pool; pages that are left behind the new end are given back (one reference less, table slot -1).
 * kept[b][i] is the old place of entry i, -1 behind the last; new_weights[b] the weights of the kept entries, 0 behind them; the other new_ arrays are
 * the old ones afterwards, and may be them.  Requests with keep entries or fewer stay as they are, and so do, reported, those with a page that would be written and is shared
 * (more than one reference: DSV4_STATUS_SHARED_PAGE) or one that is not in the pool.
 * Pools are [layers][num_pages][64][entry_bytes], entry_bytes a multiple of 16: K and V pages, and the latent cache's as well; no two of them may overlap.  scratch: 4 * B + B * max_pages * 64 int32.
 */
#define DSV4_STATUS_SHARED_PAGE 12
#define DSV4_EVICT_POOLS 4
typedef struct Dsv4KvEvictParams {
    int32_t B;
    int32_t max_pages;
    int32_t pools;
    int32_t keep;
    int32_t first;
    int32_t recent;
    int64_t num_pages;
    int64_t layers;
    const int32_t* keep_each;   /* optional int32 [B] */
    const int32_t* block_table; /* int32 [B][max_pages] */
    const int32_t* kv_len;      /* int32 [B] */
    const int32_t* refs;        /* int32 [num_pages] */
    const float*   weights;     /* float [B][weight_stride] */
    int64_t        weight_stride;   /* >= max_pages * 64 */
    int32_t*       new_table;
    int32_t*       new_len;
    int32_t*       new_refs;
    float*         new_weights;
    int32_t*       kept;        /* int32 [B][max_pages * 64] */
    int32_t*       scratch;
    int32_t*       status;
    void*          pool[DSV4_EVICT_POOLS];
    int64_t        entry_bytes[DSV4_EVICT_POOLS];
} Dsv4KvEvictParams;

int dsv4_kv_evict(const Dsv4KvEvictParams* p, void* stream);

#ifdef __cplusplus
}
#endif
#endif  /* DSV4_GQA_H_ */
