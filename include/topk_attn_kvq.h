/*
 * topk_attn_kvq.h — C ABI of the 8-bit K/V cache and of the attention of a batch behind a shared prefix (libtka.so).
 *
 *   tka_kvq_write          new K and V rows are quantised into the cache
 *   tka_kvq_read           rows of the cache as 16-bit numbers again
 *   tka_kvq_scores         stage-1 scores over 8-bit keys (what tka_topk_f32 selects from)
 *   tka_kvq_flash_decode   one decode step of attention over an 8-bit cache, all rows or the listed ones
 *   tka_prefix_decode      one decode step of a batch whose sequences share a prefix and have a suffix each
 *
 * The conventions are those of topk_attn.h: device pointers owned by the caller, asynchronous on `stream`, no
 * allocation, tka_status returned, every check before the first HIP call, reserved fields zero, 64-bit offsets.
 * `stream` and all pointers belong to the device that is current when the call is made.  A call whose rows would take
 * more than 2^32 - 1 threads gives TKA_EUNSUPPORTED.
 *
 * An 8-bit row.  The 128 elements x of one (batch entry, token, KV head) are held as 128 one-byte codes and one fp32
 * scale and stand for code * scale.  Let A = max |x|.
 *   TKA_KV_E4M3   scale = the smallest power of two with A <= 448 * scale, at least 2^-126;
 *                 code  = x / scale (exact) rounded to the nearest OCP e4m3 number, ties to even.
 *   TKA_KV_INT8   scale = max(fp32(A / 127), 2^-126);  code = x * min(fp32(127 / A), 2^126) in fp32, rounded to the
 *                 nearest whole number, ties to even (-127 .. 127).
 * A row that holds an infinity or a NaN gets scale = NaN and codes 0: it reads back as NaN and shows wherever it is used.
 * The readers accept any code byte and any fp32 scale: they need not come from tka_kvq_write.  (The attention multiplies a key
 * row's scale by the call's scale * log2 e first: a product beyond fp32's range counts as infinite.)
 */
#ifndef TOPK_ATTN_KVQ_H_
#define TOPK_ATTN_KVQ_H_

#include "topk_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum tka_kv_format {
  TKA_KV_16BIT = 0, /* rows of 16-bit numbers of the call's dtype, no scales (tka_prefix_decode only) */
  TKA_KV_E4M3 = 1,
  TKA_KV_INT8 = 2
} tka_kv_format;

/* Keys and values of `batch` entries x `rows` tokens x `num_kv_heads` heads.  Row (b,t,h) of the keys starts at
 * k + (b*stride_b + t*stride_n + h*stride_h) elements (one byte each in the 8-bit formats, two in TKA_KV_16BIT), its scale
 * is k_scale[b*scale_stride_b + t*scale_stride_n + h*scale_stride_h]; values likewise with the same strides.  Rows are
 * 16-byte aligned.  Tokens that lie next to each other in a head's scales (scale_stride_n = 1) are what the kernels
 * read best; codes may lie token by token or head by head.  The attention entry points take rows of a head, and
 * scales, up to 64 MiB apart (TKA_EUNSUPPORTED beyond). */
typedef struct tka_kv_cache {
  void* k;
  void* v;                /* may be NULL where only keys are read (tka_kvq_scores)              */
  float* k_scale;         /* NULL in TKA_KV_16BIT                                               */
  float* v_scale;
  int32_t format;         /* tka_kv_format                                                      */
  int32_t batch;
  int32_t num_kv_heads;
  int32_t head_dim;       /* must be 128                                                        */
  int64_t rows;           /* tokens per entry there is room for, <= 2^31 - 1025                 */
  int64_t stride_b, stride_n, stride_h;
  int64_t scale_stride_b, scale_stride_n, scale_stride_h;
} tka_kv_cache;

/* Row (b,t,h) of the inputs goes to row (b, start[b] + t, h) of the cache for t < count[b].  Rows of the cache that get
 * none keep what they hold; a target outside [0, rows) is dropped, counts are taken between 0 and num_tokens.  The rows of
 * the cache must be disjoint: its strides have to nest (each at least the extent of the smaller ones). */
typedef struct tka_kvq_write_args {
  tka_kv_cache cache;
  const void* k;          /* device; row (b,t,h) at k + b*stride_b + t*stride_n + h*stride_h, 16-byte aligned */
  const void* v;          /* device; same strides                                               */
  int32_t dtype;          /* tka_dtype of k and v                                               */
  int32_t num_tokens;
  int64_t stride_b, stride_n, stride_h;
  const int32_t* start;   /* device [batch]; NULL = 0                                           */
  const int32_t* count;   /* device [batch]; NULL = num_tokens                                  */
  void* stream;
} tka_kvq_write_args;

int tka_kvq_write(const tka_kvq_write_args* args);

/* Row (b, start[b] + t, h) of the cache goes to row (b,t,h) of the outputs for t < count[b], as code * scale (fp32)
 * rounded to `dtype`, numbers beyond its range as its largest.  Output rows without a source (behind count[b], or from
 * outside [0, rows)) keep what they hold; output rows must be disjoint like those of a written cache. */
typedef struct tka_kvq_read_args {
  tka_kv_cache cache;
  void* k;                /* device; rows as in tka_kvq_write_args                              */
  void* v;
  int32_t dtype;
  int32_t num_tokens;
  int64_t stride_b, stride_n, stride_h;
  const int32_t* start;
  const int32_t* count;
  void* stream;
} tka_kvq_read_args;

int tka_kvq_read(const tka_kvq_read_args* args);

/* scores[b][h][t] = (dot * k_scale) * scale for t < kv_len[b], -infinity behind it; dot = the sum of topk_attn.h's score
 * definition with the codes in the place of the keys, bit for bit (fp32, the group's queries added up first).
 * tka_topk_f32 over the scores is the exact selection; rows that are not there come last in it. */
typedef struct tka_kvq_scores_args {
  tka_kv_cache cache;     /* v and v_scale are not read                                         */
  const void* q;          /* device [batch][num_kv_heads*group][128]                            */
  int32_t dtype;          /* of q                                                               */
  int32_t group;          /* 1, 2, 4 or 8                                                       */
  int64_t q_stride_b;
  const int32_t* kv_len;  /* device [batch], taken between 0 and rows; NULL = rows              */
  float scale;
  int32_t reserved0;
  float* out_scores;      /* device [batch][num_kv_heads][rows]                                 */
  void* stream;
} tka_kvq_scores_args;

int tka_kvq_scores(const tka_kvq_scores_args* args);

/* out = softmax(scale * q.K^T) V over the rows t < kv_len[b], or over the listed rows.  A query without a row gets zeros
 * and lse = -infinity.  The entries of a list count as often as they stand in it; ids outside [0, kv_len[b]) are
 * skipped.  Value scales are held relative to the largest one that was met: beside it, what rows of much smaller scales lose
 * is below 2^-22 of the largest |value|. */
typedef struct tka_kvq_flash_decode_args {
  tka_kv_cache cache;     /* stride_b = 0: shared by the batch                                  */
  const void* q;          /* device [batch][num_kv_heads*group][128]                            */
  void* out;              /* device [batch][num_kv_heads*group][128]                            */
  int32_t dtype;          /* of q                                                               */
  int32_t out_dtype;
  int32_t group;          /* 1, 2, 4 or 8                                                       */
  int32_t num_splits;     /* workgroups per (batch entry, KV head); 0 = choose                  */
  int64_t q_stride_b;
  int64_t out_stride_b;
  const int32_t* kv_len;  /* device [batch]; NULL = rows                                        */
  const int32_t* kv_idx;  /* device [batch][num_kv_heads][idx_len] or NULL                      */
  const int32_t* kv_count;/* device [batch][num_kv_heads] or NULL = idx_len; needs kv_idx       */
  int32_t idx_len;
  float scale;
  float* out_lse;         /* device [batch][num_kv_heads*group] natural-log LSE; may be NULL    */
  void* workspace;
  size_t workspace_bytes;
  void* stream;
} tka_kvq_flash_decode_args;

size_t tka_kvq_flash_decode_workspace_bytes(const tka_kvq_flash_decode_args* args);
int tka_kvq_flash_decode(const tka_kvq_flash_decode_args* args);

/* out[b] = softmax(scale * q[b].K^T) V over the rows of the prefix followed by the first suffix_len[b] rows of suffix
 * entry b: the prefix is read once for the whole batch.  Both caches have one format; `prefix.batch` is 1, `suffix.batch`
 * is the batch.  A prefix without rows (prefix.rows = 0) is allowed (its pointers are then not read), and so is a suffix
 * without rows (suffix.rows = 0, suffix.batch still the batch).  Value scales as in tka_kvq_flash_decode. */
typedef struct tka_prefix_decode_args {
  tka_kv_cache prefix;
  tka_kv_cache suffix;
  const void* q;          /* device [batch][num_kv_heads*group][128]                            */
  void* out;
  int32_t dtype;          /* of q, and of the caches in TKA_KV_16BIT                            */
  int32_t out_dtype;
  int32_t group;          /* 1, 2, 4 or 8                                                       */
  int32_t num_splits;     /* of the prefix; 0 = choose                                          */
  int64_t q_stride_b;
  int64_t out_stride_b;
  const int32_t* suffix_len; /* device [batch], taken between 0 and suffix.rows; NULL = suffix.rows */
  float scale;
  int32_t reserved0;
  float* out_lse;
  void* workspace;
  size_t workspace_bytes;
  void* stream;
} tka_prefix_decode_args;

size_t tka_prefix_decode_workspace_bytes(const tka_prefix_decode_args* args);
int tka_prefix_decode(const tka_prefix_decode_args* args);

/* Testing hook (process-wide): tka_prefix_decode takes 16 * row_tiles query rows (1, 2, 4, 8, 16; 16-bit rows: up to 4) with each
 * tile of the prefix in place of the number it would choose, 0 = choose.  Results stay within the same error bounds. */
int tka_kvq_test_row_tiles(int32_t row_tiles);

#ifdef __cplusplus
}
#endif

#endif /* TOPK_ATTN_KVQ_H_ */
