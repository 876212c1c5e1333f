/*
 * oscar_operators.h -- C ABI of the operators around the OSCAR INT2 cache that have no
 * counterpart in the reference, beside oscar_amd.h and in its manner: device pointers,
 * strides, shapes and a HIP stream passed as void*; arguments are validated on the host;
 * launches are asynchronous on `stream`; nothing is allocated; 0 or a negative errno-style
 * status is returned, with the message in oscar_last_error().
 *
 * All entry points but oscarop_decode_step_v1 may be captured into a HIP graph, with a
 * workspace that nothing else uses while the graph may be replayed.
 */
#ifndef OSCAR_OPERATORS_H
#define OSCAR_OPERATORS_H

#include "oscar_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- attention scores ----------------------------------------------------------------
 * The score of key t for a query at position p (0-based in its request) and head h, where
 * s = scale q.k is the plain one:
 *   s' = soft_cap tanh(s / soft_cap) + alibi_slopes[h] (t - p)
 * soft_cap 0 leaves s as it is, a NULL alibi_slopes adds nothing.  Keys a query does not
 * see stay unseen whatever their score. */
typedef struct oscarop_score_v1 {
  float soft_cap;               /* 0, or in [2^-20, 1024] */
  const float* alibi_slopes;    /* [num_q_heads] fp32 device, or NULL */
} oscarop_score_v1;

/* oscar_attn_decode_v1, oscar_attn_prefill_v1 and oscar_decode_step_v1 with these scores
 * (score == NULL, or no cap and no slopes: the plain calls).  out, lse and every rule of
 * the plain calls are the same otherwise, their roundings included: history values are
 * q_dtype(fp16(x)), but V is unrounded in the decode's tiles without window copies or current
 * keys; there the probabilities times V's scale are rounded to fp16, in its other tiles the
 * probabilities to two parts in the queries' type, in the prefill to fp16; sums and the softmax
 * are fp32.  A capped score keeps soft_cap 2^-22.  The decode's waves take an item's tiles as they get to them, so
 * that its last bits may differ from run to run where an item has several tiles. */
int oscarop_attn_decode_v1(const oscar_attn_args_v1* args, const oscarop_score_v1* score, void* stream);
int oscarop_attn_prefill_v1(const oscar_prefill_args_v1* args, const oscarop_score_v1* score, void* stream);
int oscarop_decode_step_v1(oscar_context_v1* ctx, oscar_step_args_v1* args, const oscarop_score_v1* score, void* stream);

/* ---- RMS norm of every query and key head with the position rotation ----------------
 * For each row x of head_dim values (a token's head):
 *   y = x / sqrt(mean(x^2) + eps) * (w + weight_offset)     (a NULL weight: no gain, and no
 *                                                            offset either)
 * then, over its first rotary_dim values, pairs (a, b) turn by the token's angles:
 *   (a, b) -> (a cos - b sin, b cos + a sin),
 * a pair being (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when interleaved.  fp32
 * throughout, rounded once to the rows' type. */
typedef struct oscarop_norm_rope_args_v1 {
  const void* q;                /* [num_tokens, num_q_heads, head_dim] */
  int64_t q_stride_token;       /* elements; heads are head_dim apart */
  int64_t num_q_heads;          /* 0: no queries */
  const void* k;                /* [num_tokens, num_kv_heads, head_dim] */
  int64_t k_stride_token;
  int64_t num_kv_heads;         /* 0: no keys */
  int64_t num_tokens;
  int64_t head_dim;             /* 128 or 256 */
  int32_t dtype;                /* enum oscar_dtype of q, k and the outputs */
  const void* q_weight;         /* [head_dim], or NULL: no gain */
  const void* k_weight;
  int32_t weight_dtype;
  float weight_offset;          /* added to the weights: 1 for those stored around zero */
  float eps;
  const void* positions;        /* [num_tokens] device */
  int32_t positions_int64;      /* 0: int32 */
  /* [cos_sin_rows, rotary_dim], contiguous: row p holds the rotary_dim / 2 cosines of
   * position p, then its sines.  A token whose position lies outside [0, cos_sin_rows)
   * gets NaN rows. */
  const void* cos_sin;
  int32_t cos_sin_dtype;
  int32_t interleaved;
  int64_t cos_sin_rows;
  int64_t rotary_dim;           /* a multiple of 16, <= head_dim */
  /* outputs; q_out == q and k_out == k (with the same strides) work in place, any other
   * overlap of inputs and outputs does not */
  void* q_out;
  int64_t q_out_stride_token;
  void* k_out;
  int64_t k_out_stride_token;
} oscarop_norm_rope_args_v1;

int oscarop_norm_rope_v1(const oscarop_norm_rope_args_v1* args, void* stream);

/* ---- the attention weight that each cached token received -----------------------------
 * weights[r][h][t] += sum over request r's queries and the query heads of KV head h of
 * exp(s' - lse), s' being the row's score of key t (unseen keys: nothing) and lse its
 * log-sum-exp as the attention call over the same batch wrote it; a row with lse = -inf
 * saw no key and adds nothing.  Keys as oscar_attn_decode_v1 reads them: request r's
 * queries are rows [query_start_loc[r], query_start_loc[r + 1]) of q, its length
 * seq_lens[r] includes the current chunk when k_new is given, and query i of n_q sees keys
 * [0, seq - n_q + i + 1).  With history 0 and k_new the rows may be unrotated ones.  No
 * rounding below fp32.  The order of the sums follows from the call's sizes alone (num_reqs,
 * heads, max_seq_len, max_query_len, weights_cols): the same call gives the same bits, a
 * request in a call of other sizes may differ by fp32 roundings.  A request that does not fit
 * (queries past num_tokens, a length past weights_cols, a history past the block table)
 * reads nothing and its weights become NaN. */
typedef struct oscarop_weights_args_v1 {
  const void* q;                /* [num_tokens, num_q_heads, D] in q_dtype */
  int64_t num_tokens;           /* at most 2^24 */
  int64_t num_q_heads;
  int64_t q_stride_token;       /* elements */
  const void* k_new;            /* [num_tokens, Hk, D] current chunk, or NULL (cache only) */
  int64_t k_new_stride_token;
  oscar_cache_v1 cache;         /* the v side is not read */
  const int32_t* block_table;   /* [block_table_rows, block_table_cols] */
  int64_t block_table_stride;
  int64_t block_table_rows;
  int64_t block_table_cols;
  const int32_t* query_start_loc; /* device [num_reqs + 1] */
  const int32_t* seq_lens;        /* device [num_reqs] */
  int32_t num_reqs;
  int32_t q_dtype;              /* OSCAR_BF16 or OSCAR_F16 */
  /* the longest length and the most queries of a request: they size the launch; requests past
   * them are served as well */
  int64_t max_seq_len;          /* at most 2^30, as weights_cols */
  int64_t max_query_len;        /* at most 2^24 */
  const oscar_staging_v1* staging; /* NULL = no window; its v side is not read */
  float scale;
  const float* lse;             /* [num_tokens, num_q_heads] */
  float* weights;               /* [num_reqs][Hk][weights_cols], strides in elements */
  int64_t weights_stride_request;
  int64_t weights_stride_head;
  int64_t weights_cols;
  void* workspace;              /* >= oscarop_attn_weights_workspace_bytes_v1(args), 16-byte aligned */
  int64_t workspace_bytes;
} oscarop_weights_args_v1;

/* reads the sizes of *args alone; -22 for sizes that the call would refuse */
int64_t oscarop_attn_weights_workspace_bytes_v1(const oscarop_weights_args_v1* args);
int oscarop_attn_weights_v1(const oscarop_weights_args_v1* args, const oscarop_score_v1* score, void* stream);

/* ---- eviction by accumulated weight ----------------------------------------------------
 * Of request r's tokens [sink, tail) the `drop` of least weight leave the cache, for each KV
 * head its own (equal weights: the later token first; NaN counts as the largest).  The kept
 * tokens of [tail - drop, tail) move into the places of the dropped ones of
 * [sink, tail - drop), the i-th into the i-th, with slot bytes and weights; a place that is
 * written loses its FP32 window copy.  The tokens [tail, seq) stay in their pages, so that
 * with tail and drop whole pages the request's pages [(tail - drop) / block_size,
 * tail / block_size) are free afterwards and its length is seq - drop: the caller takes them
 * out of the block table (the call leaves it alone, since the layers of a model share it).
 * No page of [sink, tail) may belong to another request or come twice. */
typedef struct oscarop_evict_args_v1 {
  const float* weights;         /* [num_reqs][Hk][weights_cols], strides in elements */
  int64_t weights_stride_request;
  int64_t weights_stride_head;
  int64_t weights_cols;
  /* the weights by new position, zero from the new length on; no overlap with weights */
  float* weights_out;
  int64_t out_stride_request;
  int64_t out_stride_head;
  oscar_cache_v1 cache;
  const int32_t* block_table;   /* [block_table_rows, block_table_cols] */
  int64_t block_table_stride;
  int64_t block_table_rows;
  int64_t block_table_cols;
  /* device [num_reqs][4]: seq, sink, tail, drop.  A request that does not fit (0 <= sink,
   * 0 <= drop <= tail - sink, tail <= seq <= weights_cols, drop <= max_drop, pages within
   * the table) keeps its cache, and its weights are copied. */
  const int32_t* requests;
  int32_t num_reqs;
  int32_t reserved;
  int64_t max_drop;             /* the largest drop: whole pages */
  const oscar_staging_v1* staging; /* NULL = no window; only its owner tags are used */
  void* workspace;              /* >= oscarop_evict_workspace_bytes_v1(...), 16-byte aligned */
  int64_t workspace_bytes;
} oscarop_evict_args_v1;

/* -22 for sizes that the call would refuse: num_reqs or num_kv_heads past 65535, 2^30 or
 * more tokens to drop, more bytes than an int64_t counts */
int64_t oscarop_evict_workspace_bytes_v1(int64_t num_reqs, int64_t num_kv_heads, int64_t max_drop);
int oscarop_evict_v1(const oscarop_evict_args_v1* args, void* stream);

/* ---- pages and slots of a step's tokens -------------------------------------------------
 * Request r has lengths[r] tokens in the cache and counts[r] (below 1: none) rows of the
 * step, next to the rows of the request before it.  All of its rows, or those with a mark in
 * `keep`, take the places lengths[r], lengths[r] + 1, ... in their order.  Pages that the table does
 * not have yet come off the top of the pool, requests in their order: a request gets all of its
 * pages if it needs none, or if they and those of the requests before it are in the pool
 * (refused requests' pages count as well), and none otherwise.
 *   query_start_loc[r]  its first row       slots[i]      page * block_size + offset of the row's
 *   seq_lens[r]         its length after           place; -1 without a mark, for a request
 *   granted[r]          whether it has             that was refused, behind the last request,
 *                       its pages                  and where the table holds a negative page
 *   positions[i]        lengths[r] + the row's number in its request; 0 behind the last one
 * and the new pages are in block_table, their number off *pool_count.  A request that does not
 * fit (a negative length, rows past num_tokens, an end past the table or 2^31) is refused as
 * well, without counting.  Query starts stay within num_tokens.  No overlap of any two
 * arrays. */
typedef struct oscarop_map_args_v1 {
  const int32_t* lengths;       /* [num_reqs] device, as all arrays */
  const int32_t* counts;        /* [num_reqs] */
  const uint8_t* keep;          /* [num_tokens], nonzero: a mark; or NULL */
  int32_t num_reqs;             /* at most 65536 */
  int32_t block_size;           /* tokens per page */
  int64_t num_tokens;           /* rows of the step, at most 2^30 (65536 with keep) */
  int32_t* block_table;         /* [block_table_rows, block_table_cols] */
  int64_t block_table_stride;
  int64_t block_table_rows;     /* at least num_reqs */
  int64_t block_table_cols;
  const int32_t* pool_pages;    /* [pool_size]: the first *pool_count are free */
  int32_t* pool_count;
  int64_t pool_size;
  int32_t* query_start_loc;     /* [num_reqs + 1] */
  int32_t* seq_lens;            /* [num_reqs] */
  int64_t* slots;               /* [num_tokens] */
  int64_t* positions;           /* [num_tokens] */
  uint8_t* granted;             /* [num_reqs] */
  void* workspace;              /* >= oscarop_map_workspace_bytes_v1(...), 4-byte aligned */
  int64_t workspace_bytes;
} oscarop_map_args_v1;

/* -22 for sizes that the call would refuse */
int64_t oscarop_map_workspace_bytes_v1(int64_t num_reqs, int64_t num_tokens, int32_t keep);
int oscarop_map_v1(const oscarop_map_args_v1* args, void* stream);

/* The pages of request r behind new_lengths[r], ceil(new / block_size) up to
 * ceil(lengths[r] / block_size), go back on top of the pool, requests in their order (what
 * oscarop_map_v1 took last comes to lie as it lay).  The table keeps them.  A request with a
 * new length below 0 or above its length, or with pages past the table, gives none, nor do the
 * first one that the pool has no room for and those with pages behind it. */
typedef struct oscarop_release_args_v1 {
  const int32_t* lengths;       /* [num_reqs] device, as all arrays */
  const int32_t* new_lengths;   /* [num_reqs] */
  int32_t num_reqs;             /* at most 65536 */
  int32_t block_size;
  const int32_t* block_table;
  int64_t block_table_stride;
  int64_t block_table_rows;
  int64_t block_table_cols;
  int32_t* pool_pages;          /* [pool_size] */
  int32_t* pool_count;
  int64_t pool_size;
} oscarop_release_args_v1;

int oscarop_release_v1(const oscarop_release_args_v1* args, void* stream);

/* ---- ancestor masks of drafted trees ----------------------------------------------------
 * Node i of request r is row query_start_loc[r] + i; parents holds each node's parent as a
 * node of its request (-1: a root), which comes before it.  Bit j mod 64 of word j / 64 of a
 * row of mask: node j is the row's node or one of its ancestors; depths: the number of
 * these.  A node whose parent is no earlier one (nor -1), and all below it, has no bit and
 * depth -1, as have the nodes of a request of more than max_nodes, and rows of no request. */
typedef struct oscarop_tree_args_v1 {
  const int32_t* parents;         /* [num_tokens] device, as all arrays */
  const int32_t* query_start_loc; /* [num_reqs + 1] */
  int32_t num_reqs;               /* at most 65535 */
  int32_t max_nodes;              /* of a request, at most 1024 */
  int64_t num_tokens;             /* at most 2^30 */
  int64_t* mask;                  /* [num_tokens][mask_words] */
  int64_t mask_words;             /* ceil(max_nodes / 64) */
  int32_t* depths;                /* [num_tokens] */
} oscarop_tree_args_v1;

int oscarop_tree_mask_v1(const oscarop_tree_args_v1* args, void* stream);

/* ---- attention of drafted trees over the INT2 history -----------------------------------
 * oscarop_attn_decode_v1 for chunks whose rows see each other by a mask: query i of n_q sees
 * all of the history, and chunk row j <= i if bit j of its row of mask is set (rows past the
 * mask's words are not seen).  A row that sees no key gets zeros and lse -inf.  No
 * alibi_slopes (a node's distance is its depth, not its row); scale > 0.  History keys are
 * q_dtype(fp16(x)), history values fp16(x), the chunk's as they are; probabilities are rounded to
 * fp16 for the history and an fp16 chunk, to two bf16 parts for a bf16 one; sums and the softmax are fp32,
 * and no sum of finite values overflows (chunks of up to 2^17 rows).  The same plan gives the same bits. */
#define OSCAROP_TREE_ITEM_INTS 12

typedef struct oscarop_tree_sizes_v1 {
  int32_t num_items;
  int32_t num_groups;
  int64_t partial_rows;
  int64_t partial_bytes;        /* workspace of the call */
} oscarop_tree_sizes_v1;

/* Host plan, as oscar_attn_plan_v1: query starts [num_reqs + 1] and lengths (with the chunk);
 * items [OSCAROP_TREE_ITEM_INTS] and groups [OSCAR_GROUP_INTS] each, which the caller copies to
 * the device.  Returns the number of items, -28 with the sizes in *plan if the buffers are too
 * small; items or groups NULL: only the sizes. */
int oscarop_tree_plan_v1(const int32_t* qsl, const int32_t* seqs, int32_t num_reqs, int32_t num_kv_heads, int32_t group,
                         int32_t head_dim, int32_t target_items, int32_t* items, int32_t max_items, int32_t* groups,
                         int32_t max_groups, oscarop_tree_sizes_v1* plan);

typedef struct oscarop_tree_attn_args_v1 {
  oscar_attn_args_v1 attn;      /* as the decode's; items and groups are the tree plan's, phases 0 */
  const int64_t* mask;          /* [num_tokens][mask_words] */
  int64_t mask_words;
  int64_t partial_rows;         /* the plan's */
} oscarop_tree_attn_args_v1;

int oscarop_attn_tree_v1(const oscarop_tree_attn_args_v1* args, const oscarop_score_v1* score, void* stream);

/* ---- bounds of the keys of each page ----------------------------------------------------
 * bounds[page][h][0 / 1][d]: the least / largest of the page's keys fp16(code * scale + zero)
 * over the tokens that it holds (NaN if one of them is), for the pages of request r's columns
 * [lengths[r] / block_size, ceil(seq_lens[r] / block_size)) where seq_lens[r] > lengths[r]; all
 * others stay.  Keys of the FP32 window count as their slots hold them.  A request with a
 * negative length or columns past the table, and pages outside the cache, are left alone.
 * No page may come twice. */
typedef struct oscarop_bounds_args_v1 {
  oscar_cache_v1 cache;           /* the v side is not read */
  const int32_t* block_table;
  int64_t block_table_stride;
  int64_t block_table_rows;
  int64_t block_table_cols;
  const int32_t* lengths;         /* [num_reqs] device: tokens before */
  const int32_t* seq_lens;        /* [num_reqs] device: and after */
  int32_t num_reqs;               /* at most 65535, as KV heads */
  int32_t reserved;
  int64_t max_new;                /* the most new tokens of a request: sizes the launch (0: none); pages
                                     of a request that grew by more take turns */
  void* bounds;                   /* fp16 [num_blocks][Hk][2][D], 16-byte aligned */
} oscarop_bounds_args_v1;

int oscarop_page_bounds_v1(const oscarop_bounds_args_v1* args, void* stream);

/* ---- pages that promise the largest scores ----------------------------------------------
 * Request r has n_q queries and a history of h tokens (seq_lens[r], less n_q with has_new)
 * in P = ceil(h / block_size) pages.  With P <= budget all of them are chosen, otherwise the first
 * first_pages, the last last_pages and of the others those of the largest score (equal
 * scores: the earlier page first; a score of a bound or a query that is not finite counts as the
 * largest), budget in all, for each KV head its own.  A page's score: the largest, over the request's queries and the query
 * heads of the KV head, of the sum over the channels of max(q low, q high), summed in 64
 * bits.  table[r][h] holds the chosen pages in ascending order of their columns and
 * pages[r][h] these columns, -1 behind them.  A request that does not fit (queries past
 * num_tokens, a negative history, columns past the table) gets -1 throughout.  Without has_new
 * the queries have to lie in the last last_pages pages for the attention to know what each sees. */
#define OSCAROP_SELECT_ARRIVAL 32 /* int32 of a list's arrival counter: a cache line of its own */
typedef struct oscarop_select_args_v1 {
  const void* q;                  /* [num_tokens, num_q_heads, D] in q_dtype */
  int64_t num_tokens;
  int64_t num_q_heads;
  int64_t q_stride_token;         /* elements, a multiple of 8; rows 16-byte aligned */
  int32_t q_dtype;                /* OSCAR_BF16 or OSCAR_F16 */
  int32_t has_new;
  const void* bounds;             /* as oscarop_page_bounds_v1 leaves them */
  int64_t num_blocks;
  int64_t num_kv_heads;           /* at most 65535 */
  int64_t head_dim;               /* 128 or 256 */
  int64_t block_size;
  const int32_t* block_table;
  int64_t block_table_stride;
  int64_t block_table_rows;
  int64_t block_table_cols;
  const int32_t* query_start_loc; /* [num_reqs + 1] device */
  const int32_t* seq_lens;        /* [num_reqs] device */
  int32_t num_reqs;               /* at most 65535 */
  int32_t max_pages;              /* the most pages of a history: sizes the launch */
  int32_t budget;                 /* at least first_pages + last_pages + 1 */
  int32_t first_pages;            /* >= 0 */
  int32_t last_pages;             /* >= 1 */
  int32_t reserved;
  int32_t* table;                 /* [num_reqs][Hk][budget] */
  int32_t* pages;                 /* [num_reqs][Hk][budget], or NULL */
  void* workspace;                /* >= oscarop_select_workspace_bytes_v1(args), 16-byte aligned */
  int64_t workspace_bytes;
  /* [num_reqs * Hk][OSCAROP_SELECT_ARRIVAL], of which the first is used, zero before the first
   * call; each call leaves them zero.  As the workspace, nothing else uses them while a call runs.
   * Not read if no history exceeds the budget. */
  int32_t* arrivals;
} oscarop_select_args_v1;

/* reads the sizes of *args alone; -22 for sizes that the call would refuse */
int64_t oscarop_select_workspace_bytes_v1(const oscarop_select_args_v1* args);
int oscarop_select_v1(const oscarop_select_args_v1* args, void* stream);

/* oscarop_attn_decode_v1 with a block table for each KV head: head h of request r reads row
 * r of block_table shifted by h * table_stride_head, as oscarop_select_v1 writes it.  The
 * lengths and the plan are those of the chosen tokens.  History keys are q_dtype(fp16(x)), history
 * values fp16(x) (full tiles of codes: x itself), the chunk's as they are; probabilities are rounded to
 * fp16 times a value's scale in full tiles of codes, to two parts in q_dtype elsewhere; sums and the softmax
 * are fp32 and hold probabilities of up to 2^8, as the decode's: with n keys, values of the chunk beyond
 * 1e36 / n can overflow them.  A value that is not finite reaches no query that does not see its token.  No alibi_slopes (the chosen pages' distances are
 * not the table's); scale > 0. */
int oscarop_attn_selected_v1(const oscar_attn_args_v1* args, const oscarop_score_v1* score, int64_t table_stride_head,
                             void* stream);

#ifdef __cplusplus
}
#endif
#endif /* OSCAR_OPERATORS_H */
