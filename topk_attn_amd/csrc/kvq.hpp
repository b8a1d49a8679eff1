// Parameter blocks and launch functions of the 8-bit K/V cache and of the shared-prefix attention (internal).
#pragma once
#include "../../include/topk_attn_kvq.h"
#include "common.hpp"

namespace tka {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Strides of code rows are in BYTES, those of scales in elements; a stride of 0 shares the cache among the batch.
struct KvRows {
  const unsigned char* k;
  const unsigned char* v;
  const float* ks;
  const float* vs;
  int64_t stride_b, stride_n, stride_h;
  int64_t scale_b, scale_n, scale_h;
  int64_t rows;
};

// tka_kvq_write / tka_kvq_read: `in` side and `cache` side of the copy (the read goes the other way)
struct KvqCopyParams {
  KvRows cache;             // (its pointers are written by the write kernel)
  unsigned char* k;         // 16-bit rows; strides in bytes
  unsigned char* v;
  int64_t stride_b, stride_n, stride_h;
  const int32_t* start;
  const int32_t* count;
  int batch, num_kv_heads, num_tokens;
  int tile_log2;            // a workgroup covers 2^tile_log2 tokens of each of 32 >> tile_log2 (entry, head) pairs (set by the launcher)
};
constexpr int kCopyRows = 32;   // rows of a workgroup
// Tiles of 32 tokens of one head; calls of fewer tokens take several heads into a workgroup.
struct CopyGrid {
  int tile_log2;
  int64_t token_tiles, workgroups;
};
inline CopyGrid copy_grid(int64_t pairs, int64_t num_tokens) {
  CopyGrid g = {0, 0, 0};
  while ((1 << g.tile_log2) < kCopyRows && (1 << g.tile_log2) < num_tokens) ++g.tile_log2;
  g.token_tiles = (num_tokens + (1 << g.tile_log2) - 1) >> g.tile_log2;
  const int64_t per_wg = kCopyRows >> g.tile_log2;
  g.workgroups = g.token_tiles * ((pairs + per_wg - 1) / per_wg);
  return g;
}
int launch_kvq_write(const KvqCopyParams& p, int dtype, int format, hipStream_t stream);
int launch_kvq_read(const KvqCopyParams& p, int dtype, int format, hipStream_t stream);

struct KvqScoresParams {
  KvRows cache;
  const void* q;
  int64_t q_stride_b;
  const int32_t* kv_len;
  float* scores;
  int batch, num_kv_heads, group;
  float scale;
};
constexpr int kScoreTokens = 256;   // tokens of a workgroup (512: 95 us where 256 take 92, 1024: 102)
int launch_kvq_scores(const KvqScoresParams& p, int dtype, int format, hipStream_t stream);

// Attention over up to two sources: `shared`, whose rows every query row of the batch attends to, and `own`, whose
// entry b the queries of entry b attend to.  The grid is the shared items, then the own items.
struct KvAttendParams {
  const void* q;
  int64_t q_stride_b;
  int batch, num_kv_heads, group_log2;
  KvRows shared;
  int shared_splits;        // 0: no shared rows
  int shared_tps;           // tokens per split, a multiple of kAttendTile
  int row_blocks;           // query rows of a head (batch * group) in blocks of 16 * row_tiles
  KvRows own;
  int own_splits;           // 0: no own rows
  int own_tps;
  const int32_t* own_len;   // [batch] or nullptr
  const int32_t* kv_idx;    // [batch][num_kv_heads][idx_len] or nullptr
  const int32_t* kv_count;  // [batch][num_kv_heads] or nullptr
  int idx_len;
  int num_splits;           // partials per query row: shared_splits + own_splits
  int to_workspace;         // the launch writes partials (0: finished rows)
  f32x2* part_ml;           // [rows][num_splits] reference (base 2) and sum of the weights
  float* part_acc;          // [rows][num_splits][128], normalised
  void* out;
  float* out_lse;
  int64_t out_stride_b;
  int out_dtype;
  float scale_log2e;
};
constexpr int kAttendTile = 32;   // tokens of a wave's tile
// row_tiles: sixteens of query rows that a workgroup takes with each tile of the shared source: 1, 2, 4, in 8 bits also 8 and 16;
// 0 = the short form, one workgroup per (entry, head) and one split of each source.
int launch_kv_attend(const KvAttendParams& p, int dtype, int format, int row_tiles, hipStream_t stream);

// The own rows (one workgroup per entry and head, whatever own_splits says) joined with num_splits partials of the shared ones.
int launch_kv_attend_join(const KvAttendParams& p, int dtype, int format, hipStream_t stream);

// Joins the partials of the query rows and writes p.out / p.out_lse (num_splits > 1).
int launch_kv_combine(const KvAttendParams& p, hipStream_t stream);

}  // namespace tka
