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

#ifdef __cplusplus
}
#endif
#endif /* OSCAR_OPERATORS_H */
