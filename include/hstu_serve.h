/* C ABI of libhstu_serve.so: serving a model from kept histories, and scoring its logits, for gfx950.
 *
 *   hstu_kv_write      quantises the keys and values of new events into the pages of a cache
 *   hstu_kv_read       the values that a cache stands for
 *   hstu_cached_attn   the pointwise-SiLU attention (recml/layers/keras/hstu.py:356-390) of each
 *                      sequence's newest events over its kept keys and values
 *
 *   hstu_log_probs_fwd log probabilities of given tokens, the entropy and the largest entries of rows of logits
 *   hstu_log_probs_bwd the gradient of those for the logits
 *
 * A cache's codes are [n_pages, H, page_size, d * bits / 8] bytes, its exponents
 * [n_pages, H, (d + 31) / 32, page_size] bytes, one pair for the keys and one for the values.  A block
 * of 32 values of one (event, head) row (the row's last block may be shorter) shares the power 2^(e - 127)
 * of its exponent byte e; codes are e2m1 (bits = 4: two to a byte, the even index in the low half) or
 * e4m3 (bits = 8).  e is the smallest in [1, 252] (bits = 8: [1, 246]; no code stands for more than fp32 holds)
 * under which the block's largest magnitude rounds to a code (at most 7 or 464 times the power), so every value
 * is off by at most half of its step; values round to the nearest code, ties to the even one, past the largest
 * to the largest.  A row that holds a value which is not finite has codes of
 * zero and exponents of 255: it stands for NaN.
 *
 * Sequence b's event at place i is in row i % page_size of page page_table[b][i / page_size].  Events whose
 * page the table does not name (an entry outside [0, n_pages)) or whose place lies outside the table are
 * not written, read as zeros, and are masked in the attention.
 *
 * Plain pointers and sizes: no framework types.  Every function returns 0 or a negative HstuServeStatus; the
 * message of the last failure on the calling thread is at hstu_serve_last_error().  Work is enqueued on
 * `stream` on the current device; nothing is allocated.
 */
#ifndef HSTU_SERVE_H_
#define HSTU_SERVE_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSTU_SERVE_ABI_VERSION 1

typedef enum HstuServeStatus {
  HSTU_SERVE_OK = 0,
  HSTU_SERVE_ERR_NULL = -1,
  HSTU_SERVE_ERR_VERSION = -2,
  HSTU_SERVE_ERR_SHAPE = -4,
  HSTU_SERVE_ERR_WORKSPACE = -5,
  HSTU_SERVE_ERR_LAUNCH = -6
} HstuServeStatus;

typedef enum HstuServeDtype { HSTU_SERVE_BF16 = 0, HSTU_SERVE_FP32 = 1 } HstuServeDtype;

/* The pages of one layer.  Pointers 16-byte aligned; page_size a multiple of 32, at most 2^20; d one of 8, 16, 24, 32, 48, 64, 96,
 * 128, 192, 256; bits 4 or 8. */
typedef struct HstuKvPages {
  void* k_codes;
  void* k_scales;
  void* v_codes;
  void* v_scales;
  const int32_t* page_table;   /* [B, table_pages] */
  int32_t n_pages, page_size, table_pages;
  int32_t B, H, d, bits, reserved0;
} HstuKvPages;

/* Rows of new events: padded [B, rows_per_seq, H, d] (offsets null) or packed [total_rows, H, d], sequence b's rows
 * from offsets[b] up to offsets[b + 1] and rows_per_seq the most that one sequence has (rows past it are not looked
 * at).  The events of sequence b take the places starts[b], starts[b] + 1, ...  k and v: bf16 or fp32, the last axis
 * contiguous, row and head strides in elements, 16-byte aligned rows.  hstu_kv_write reads them, hstu_kv_read writes
 * them (rows of no sequence are left as they were). */
typedef struct HstuKvRowsArgs {
  uint32_t struct_size;   /* sizeof(HstuKvRowsArgs)    */
  uint32_t version;       /* HSTU_SERVE_ABI_VERSION    */
  HstuKvPages pages;
  const int32_t* starts;
  const int32_t* offsets;
  int64_t total_rows;
  int32_t rows_per_seq, dtype;
  void* k;
  void* v;
  int64_t k_stride_b, k_stride_t, k_stride_h;
  int64_t v_stride_b, v_stride_t, v_stride_h;
} HstuKvRowsArgs;

int hstu_kv_write(const HstuKvRowsArgs* args, void* stream);
int hstu_kv_read(const HstuKvRowsArgs* args, void* stream);

/* out[row i] = inv_n * sum_j silu(alpha q_i . k_j + pos[L - 1 + j - i] + ts_tab[bucket(ts[min(i + 1, n - 1)] - ts[j])]) v_j
 * over the places j <= i that the cache holds, n = lengths[b] (the new events included; places at or past max_len or
 * the table's end are not there), L = max_len.  The queries are the sequence's last rows: with m of them row t is at
 * place i = n - m + t; rows at places below 0 or at places that are not there are zeros.  q and out: bf16 or fp32,
 * padded or packed like the rows of HstuKvRowsArgs.  bucket: min(floor(ln(max(1, min(|dt|, 1e9))) / bucket_size),
 * ts_buckets), the attention's law.  `workspace`: hstu_cached_attn_workspace_bytes(args) bytes of device memory. */
typedef struct HstuCachedAttnArgs {
  uint32_t struct_size;   /* sizeof(HstuCachedAttnArgs) */
  uint32_t version;       /* HSTU_SERVE_ABI_VERSION     */
  HstuKvPages pages;
  const int32_t* lengths; /* [B] */
  const int32_t* offsets;
  int64_t total_rows;
  int32_t rows_per_seq, dtype;
  const void* q;
  void* out;
  int64_t q_stride_b, q_stride_t, q_stride_h;
  int64_t o_stride_b, o_stride_t, o_stride_h;
  int32_t max_len;
  float alpha, inv_n;
  int32_t pos_heads;          /* 1 or H */
  const float* pos_tab;       /* [pos_heads, 2 max_len - 1] or null */
  const int64_t* timestamps;  /* [B, max_len] or null */
  const float* ts_tab;        /* [ts_heads, ts_buckets + 1] */
  int32_t ts_heads, ts_buckets;   /* at most 128 buckets */
  float ts_bucket_size;
  int32_t reserved0;
  void* workspace;
  size_t workspace_bytes;
} HstuCachedAttnArgs;

size_t hstu_cached_attn_workspace_bytes(const HstuCachedAttnArgs* args);
int hstu_cached_attn(const HstuCachedAttnArgs* args, void* stream);

/* Of each of `rows` rows of `vocab` logits (bf16 or fp32, row stride in elements, any alignment of the type; at
 * most 2^30 of them, and of `count` tokens, a row):
 *   log_probs[row][c] = x[tokens[row][c]] - ln sum_j exp x_j; 0 where the token is negative (nothing asked), NaN where it
 *                  is past the vocabulary
 *   entropy[row]   = -sum_j p_j ln p_j (or null)
 *   top_log_probs, top_tokens: the `top` largest entries (at most 256) in falling order, ties by the lower token; NaN
 *                  comes before all others
 * A row whose sum of exponentials is not finite and positive (a NaN, +inf, nothing but -inf) has NaN for all of them.
 * stats: [rows][3], what the backward needs (or null); for a backward with g_entropy the forward has to have `entropy` too (its sum is
 * made for that alone: without it such a backward's rows are NaN).
 * The backward writes d_logits (typed like the logits) = sum over the outputs of their gradients times theirs by the
 * logits: g_tokens [rows][count], g_entropy [rows], g_top [rows][top], each or null; tokens, top_tokens and stats as the
 * forward had and left them.  The same token twice gets both gradients; negative tokens none; one past the vocabulary
 * makes its row NaN.  The forward's workspace: hstu_log_probs_workspace_bytes(args) bytes; the backward has none. */
typedef struct HstuLogProbsArgs {
  uint32_t struct_size;   /* sizeof(HstuLogProbsArgs) */
  uint32_t version;       /* HSTU_SERVE_ABI_VERSION   */
  const void* logits;
  int64_t rows, stride;
  int32_t vocab, dtype, count, top;
  const int64_t* tokens;  /* [rows][count] */
  float* log_probs;
  float* entropy;
  float* stats;
  float* top_log_probs;
  int64_t* top_tokens;
  const float* g_tokens;
  const float* g_entropy;
  const float* g_top;
  void* d_logits;
  int64_t d_stride;
  void* workspace;
  size_t workspace_bytes;
} HstuLogProbsArgs;

size_t hstu_log_probs_workspace_bytes(const HstuLogProbsArgs* args);
int hstu_log_probs_fwd(const HstuLogProbsArgs* args, void* stream);
int hstu_log_probs_bwd(const HstuLogProbsArgs* args, void* stream);

int hstu_serve_abi_version(void);
const char* hstu_serve_last_error(void);

#ifdef __cplusplus
}
#endif

#endif  /* HSTU_SERVE_H_ */
