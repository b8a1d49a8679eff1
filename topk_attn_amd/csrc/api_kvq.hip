// C ABI of the 8-bit K/V cache and of the shared-prefix attention (topk_attn_kvq.h): argument checks (before any HIP
// call), split plans, workspace layout, launches.
#include <string.h>

#include <algorithm>
#include <atomic>
#include <utility>

#include "kvq.hpp"

namespace tka {

namespace {

bool dtype_ok(int d) { return d == TKA_F16 || d == TKA_BF16; }
bool group_ok(int g) { return g == 1 || g == 2 || g == 4 || g == 8; }
bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

constexpr int64_t kMaxExtent = 1ll << 46;      // elements that a stride may span: more than any memory, and no sum of offsets passes 64 bits
constexpr int64_t kMaxItems = 0x7fffffff;      // rows of a call, partials of a call
constexpr int64_t kMaxThreads = 0xffffffff;    // of a launch
constexpr int64_t kMaxRows = 0x7fffffff - 1024;  // (positions of a tile behind the end still fit 32 bits)

bool spans_ok(int64_t count, int64_t stride) { return stride >= 0 && (count <= 1 ? stride <= kMaxExtent : stride <= kMaxExtent / (count - 1)); }
bool strides_ok(int64_t nb, int64_t nn, int64_t nh, int64_t b, int64_t n, int64_t h) { return spans_ok(nb, b) && spans_ok(nn, n) && spans_ok(nh, h); }

// Rows of `width` at b*stride_b + t*stride_n + h*stride_h are disjoint when the strides nest.
bool disjoint(int64_t width, int64_t nb, int64_t nn, int64_t nh, int64_t sb, int64_t sn, int64_t sh) {
  std::pair<int64_t, int64_t> dims[3] = {{sb, nb}, {sn, nn}, {sh, nh}};
  std::sort(dims, dims + 3);
  int64_t extent = width;
  for (const auto& d : dims) {
    if (d.second <= 1) continue;
    if (d.first < extent) return false;
    extent += (d.second - 1) * d.first;
  }
  return true;
}

// A cache: sizes, format, strides, alignment.  `values`: its values are read or written too.
int check_cache(const tka_kv_cache& c, bool values, bool allow_16bit) {
  if (c.format != TKA_KV_E4M3 && c.format != TKA_KV_INT8 && !(allow_16bit && c.format == TKA_KV_16BIT)) return TKA_EUNSUPPORTED;
  if (c.head_dim != TKA_HEAD_DIM) return TKA_EUNSUPPORTED;
  if (c.batch < 1 || c.num_kv_heads < 1 || c.rows < 1) return TKA_EINVAL;
  if (c.batch > 65535 || c.num_kv_heads > 65535 || c.rows > kMaxRows) return TKA_EUNSUPPORTED;
  if (!c.k || (values && !c.v)) return TKA_EINVAL;
  if (!strides_ok(c.batch, c.rows, c.num_kv_heads, c.stride_b, c.stride_n, c.stride_h)) return TKA_EINVAL;
  if (c.rows > 1 && c.stride_n < TKA_HEAD_DIM) return TKA_EINVAL;
  const int64_t per16 = c.format == TKA_KV_16BIT ? 8 : 16;   // elements of sixteen bytes
  if ((c.stride_b | c.stride_n | c.stride_h) & (per16 - 1)) return TKA_EINVAL;
  if (!aligned(c.k, 16) || (values && !aligned(c.v, 16))) return TKA_EINVAL;
  if (c.format != TKA_KV_16BIT) {
    if (!c.k_scale || (values && !c.v_scale)) return TKA_EINVAL;
    if (!aligned(c.k_scale, 4) || (values && !aligned(c.v_scale, 4))) return TKA_EINVAL;
    if (!strides_ok(c.batch, c.rows, c.num_kv_heads, c.scale_stride_b, c.scale_stride_n, c.scale_stride_h)) return TKA_EINVAL;
  }
  return TKA_OK;
}

KvRows rows_of(const tka_kv_cache& c) {
  const int64_t width = c.format == TKA_KV_16BIT ? 2 : 1;
  KvRows r;
  r.k = (const unsigned char*)c.k;
  r.v = (const unsigned char*)c.v;
  r.ks = c.k_scale;
  r.vs = c.v_scale;
  r.stride_b = c.stride_b * width;
  r.stride_n = c.stride_n * width;
  r.stride_h = c.stride_h * width;
  r.scale_b = c.scale_stride_b;
  r.scale_n = c.scale_stride_n;
  r.scale_h = c.scale_stride_h;
  r.rows = c.rows;
  return r;
}

// tka_kvq_write_args and tka_kvq_read_args have the same fields.
template <typename Args>
int check_copy(const Args* a, bool write) {
  if (!a) return TKA_EINVAL;
  const tka_kv_cache& c = a->cache;
  const int rc = check_cache(c, true, false);
  if (rc != TKA_OK) return rc;
  if (!a->k || !a->v || a->num_tokens < 1) return TKA_EINVAL;
  if (!dtype_ok(a->dtype)) return TKA_EUNSUPPORTED;
  if (!strides_ok(c.batch, a->num_tokens, c.num_kv_heads, a->stride_b, a->stride_n, a->stride_h)) return TKA_EINVAL;
  if ((a->stride_b | a->stride_n | a->stride_h) & 7) return TKA_EINVAL;
  if (!aligned(a->k, 16) || !aligned(a->v, 16)) return TKA_EINVAL;
  const int64_t pairs = (int64_t)c.batch * c.num_kv_heads;
  if (a->num_tokens > kMaxItems / pairs || copy_grid(pairs, a->num_tokens).workgroups > kMaxThreads / 256) return TKA_EUNSUPPORTED;
  if (write) {
    if (!disjoint(TKA_HEAD_DIM, c.batch, c.rows, c.num_kv_heads, c.stride_b, c.stride_n, c.stride_h) ||
        !disjoint(1, c.batch, c.rows, c.num_kv_heads, c.scale_stride_b, c.scale_stride_n, c.scale_stride_h))
      return TKA_EINVAL;
  } else if (!disjoint(TKA_HEAD_DIM, c.batch, a->num_tokens, c.num_kv_heads, a->stride_b, a->stride_n, a->stride_h)) {
    return TKA_EINVAL;
  }
  return TKA_OK;
}

template <typename Args>
KvqCopyParams copy_params(const Args* a) {
  KvqCopyParams p;
  p.cache = rows_of(a->cache);
  p.k = (unsigned char*)const_cast<void*>((const void*)a->k);
  p.v = (unsigned char*)const_cast<void*>((const void*)a->v);
  p.stride_b = 2 * a->stride_b;
  p.stride_n = 2 * a->stride_n;
  p.stride_h = 2 * a->stride_h;
  p.start = a->start;
  p.count = a->count;
  p.batch = a->cache.batch;
  p.num_kv_heads = a->cache.num_kv_heads;
  p.num_tokens = a->num_tokens;
  p.tile_log2 = 0;
  return p;
}

// The attention kernels address the rows and scales of a 32-token tile with 32-bit offsets.
constexpr int64_t kMaxRowBytes = 1ll << 26;
int check_row_stride(const tka_kv_cache& c) {
  if (c.rows > 1 && c.stride_n * (c.format == TKA_KV_16BIT ? 2 : 1) > kMaxRowBytes) return TKA_EUNSUPPORTED;
  return c.rows > 1 && c.format != TKA_KV_16BIT && c.scale_stride_n * 4 > kMaxRowBytes ? TKA_EUNSUPPORTED : TKA_OK;
}

int check_query(const void* q, int dtype, int group, int64_t q_stride_b, int batch, int heads) {
  if (!q) return TKA_EINVAL;
  if (!dtype_ok(dtype) || !group_ok(group)) return TKA_EUNSUPPORTED;
  const int64_t width = (int64_t)heads * group * TKA_HEAD_DIM;
  if (!spans_ok(batch, q_stride_b) || (q_stride_b & 7) || !aligned(q, 16)) return TKA_EINVAL;
  if (batch > 1 && q_stride_b < width) return TKA_EINVAL;
  if ((int64_t)batch * heads * group > kMaxItems) return TKA_EUNSUPPORTED;
  return TKA_OK;
}

int check_out(const void* out, int out_dtype, int64_t out_stride_b, int batch, int heads, int group) {
  if (!out) return TKA_EINVAL;
  if (!dtype_ok(out_dtype)) return TKA_EUNSUPPORTED;
  if (!spans_ok(batch, out_stride_b) || (out_stride_b & 7) || !aligned(out, 16)) return TKA_EINVAL;
  if (batch > 1 && out_stride_b < (int64_t)heads * group * TKA_HEAD_DIM) return TKA_EINVAL;
  return TKA_OK;
}

int check_scores(const tka_kvq_scores_args* a) {
  if (!a) return TKA_EINVAL;
  int rc = check_cache(a->cache, false, false);
  if (rc != TKA_OK) return rc;
  rc = check_query(a->q, a->dtype, a->group, a->q_stride_b, a->cache.batch, a->cache.num_kv_heads);
  if (rc != TKA_OK) return rc;
  if (!a->out_scores || a->reserved0 != 0) return TKA_EINVAL;
  const int64_t segs = (int64_t)a->cache.batch * a->cache.num_kv_heads;
  if ((a->cache.rows + kScoreTokens - 1) / kScoreTokens > kMaxThreads / 256 / segs) return TKA_EUNSUPPORTED;
  return TKA_OK;
}

// `len` positions in `want` splits of a multiple of kTps positions, `most` splits at most.
constexpr int64_t kTps = 4 * kAttendTile;   // every wave of a workgroup has a tile
void cut(int64_t len, int64_t want, int64_t most, int* splits, int* tps) {
  want = std::min(std::max<int64_t>(want, 1), most);
  int64_t per = (len + want - 1) / want;
  per = (per + kTps - 1) / kTps * kTps;
  *splits = (int)((len + per - 1) / per);
  *tps = (int)per;
}

int log2_of(int group) { return group == 8 ? 3 : group >> 1; }

struct Plan {
  int row_tiles, row_blocks;
  int shared_splits, shared_tps, own_splits, own_tps;
  bool join_own;   // the own rows are attended to by the launch that joins the partials of the shared ones
  int parts() const { return row_tiles ? shared_splits + (join_own ? 0 : own_splits) : 1; }
  bool to_workspace() const { return parts() > 1 || join_own; }
};

// Decodes of up to this many positions per (entry, head) take one launch of one workgroup each instead of a split and a join
// (one sequence, 8 heads, group 4: 6.4 against 7.9 us at 256 positions, 8.6 against 7.8 at 512; host-bound below).
constexpr int64_t kSoloLen = 256;

// Splits of each (entry, head) of a decode.  Two workgroups a CU read best (4 x 8 x 32768 rows of e4m3: 256 workgroups 61 us, 512 45, 768
// 47, 1024 51), but between 256 and 448 pairs, which fill the CUs unevenly, four splits each (320 pairs x 8000 rows: 131 -> 112 us,
// 384 pairs 139 -> 135; 512 pairs in one split 168, in four 176).  Short calls save the second launch with one split: 32 pairs x 300
// rows 7.8 -> 7.2 us (600: 8.0 -> 10.3), 128 x 600 12.0 -> 10.5 (1200: 15.0 -> 18.3), 256 x 1200 19.7 -> 19.4 (2400: 30.9 -> 33.3).
int64_t decode_splits(int64_t segs, int64_t len) {
  if (len <= std::max<int64_t>(384, std::min<int64_t>(6 * segs, 1280))) return 1;
  return segs > 256 && segs < 448 ? 4 : 512 / segs;
}

Plan plan_decode(const tka_kvq_flash_decode_args* a) {
  Plan p = {1, 0, 0, 0, 0, 0, false};
  const int64_t segs = (int64_t)a->cache.batch * a->cache.num_kv_heads;
  const int64_t len = a->kv_idx ? a->idx_len : a->cache.rows;
  if (!a->num_splits && len <= kSoloLen) {
    p.row_tiles = 0;
    cut(len, 1, 1, &p.own_splits, &p.own_tps);
    return p;
  }
  cut(len, a->num_splits ? a->num_splits : decode_splits(segs, len), TKA_MAX_SPLITS, &p.own_splits, &p.own_tps);
  return p;
}

// Query rows of a head that a workgroup takes with each tile of the prefix, in sixteens.  More of them save reads of the rows (of the
// L2 and the memory-side cache: the blocks of a head run side by side) and conversions, fewer start and end sooner and leave the
// CU to more workgroups, so the rule goes by the size of the products, query rows x heads x positions.  Times by sixteens 1 / 2 / 4 /
// 8 / 16 in us, suffixes of 100:
//   16 x 8 x 4 (64 rows), 1000 positions    16 bit  0.5 M   10.6 / 10.9 / 16.2 / 13.4 / 13.9
//   10 x 8 x 4 (40), 8192                   int8    2.6 M   16.8 / 17.5 / 19.5 / 20.3 / 21.3
//   16 x 8 x 4, 8192                        16 bit  4.2 M   20.8 / 18.7 / 24.0 / 27.0 / 26.5
//   32 x 8 x 4 (128), 8192                  16 bit  8.4 M   30.4 / 23.4 / 27.4 / 35.6 / 31.6
//   16 x 8 x 4, 32768                       16 bit   17 M   57.1 / 40.9 / 41.5 / 55.5 / 59.1
//   32 x 8 x 4, 16384                       e4m3     17 M   38.6 / 30.0 / 32.8 / 34.9 / 33.9
//   32 x 8 x 4, 32768                       16 bit   34 M   92.6 / 57.3 / 47.2 / 61.8 / 62.1
//   32 x 8 x 4, 32768                       e4m3     34 M      - / 44.8 / 47.0 / 48.1 / 46.2
//   64 x 8 x 8 (512), 8192                  e4m3     34 M      - / 49.5 / 53.0 / 50.0 / 44.5
//   20 x 8 x 4 (80), 100000                 int8     64 M      -  / 101 /  119 / 91.3 / 96.3
//   64 x 8 x 8, 32768                       16 bit  134 M      -  / 206 /  130 /  129 /  131
//   64 x 8 x 8, 32768                       e4m3    134 M      -  / 133 /  135 /  107 / 97.0
int prefix_row_tiles(int64_t query_rows, int64_t positions, bool wide16) {
  const int64_t work = query_rows * positions;
  if (query_rows <= 16 || work <= 5 << 19) return 1;
  if (query_rows <= 32 || work <= (wide16 ? 17 << 20 : query_rows <= 128 ? 44 << 20 : 28 << 20)) return 2;
  if (wide16 || query_rows <= 64) return 4;   // (16-bit rows have no conversion to share: blocks of 128 and 256 do not win)
  return query_rows <= 128 ? 8 : 16;
}

// Short calls: one workgroup per (entry, head) attends to prefix and suffix and writes the result; the prefix is then read, and widened,
// for each entry.  Against the split form, us: 4 x 2 x 4 over 250 + 50 rows of 16 bits 7.0 and 7.7 (400 + 50: 8.6 and 7.7), 16 x 8 x 4 over
// 250 + 50 7.3 and 8.4, 64 x 16 x 4 over 250 + 20 23.5 and 17.2; 8 bits: 32 x 8 x 4 over 250 + 20 7.5 and 10.1, 64 x 8 x 8 over 400 + 100
// 16.7 and 19.6, but 4 x 8 x 4 over 400 + 50 8.3 and 7.9.
bool prefix_in_one(int64_t segs, int64_t len, bool wide16) {
  if (wide16) return segs <= 256 && len <= 320;
  return len <= 320 || (segs >= 192 && len <= 512);
}

std::atomic<int> g_row_tiles{0};   // tka_kvq_test_row_tiles

Plan plan_prefix(const tka_prefix_decode_args* a) {
  Plan p = {1, 0, 0, 0, 0, 0, false};
  const int64_t heads = a->prefix.num_kv_heads, batch = a->suffix.batch, query_rows = batch * a->group;
  const int hook = g_row_tiles.load(std::memory_order_relaxed);
  const bool wide16 = a->prefix.format == TKA_KV_16BIT;
  if (!a->num_splits && !hook && prefix_in_one(heads * batch, a->prefix.rows + a->suffix.rows, wide16)) {
    p.row_tiles = 0;
    if (a->prefix.rows) cut(a->prefix.rows, 1, 1, &p.shared_splits, &p.shared_tps);
    if (a->suffix.rows) cut(a->suffix.rows, 1, 1, &p.own_splits, &p.own_tps);
    return p;
  }
  if (a->prefix.rows) {
    p.row_tiles = hook ? (wide16 ? std::min(hook, 4) : hook) : prefix_row_tiles(query_rows, heads * a->prefix.rows, wide16);
    p.row_blocks = (int)((query_rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles));
    // One workgroup a CU for 16-bit rows and the blocks that fill a CU, two for 8-bit rows (16 x 8 x 4 over 8192 rows of 16 bits with 512
    // workgroups 21.1 us, with 256 18.7; 32768 rows of e4m3 32.8 and 34.8, with 1024 41.1).
    cut(a->prefix.rows, a->num_splits ? a->num_splits : (wide16 || p.row_tiles == 4 || p.row_tiles == 16 ? 256 : 512) / (heads * p.row_blocks), TKA_MAX_SPLITS / 2, &p.shared_splits, &p.shared_tps);
  }
  // The blocks of 256 query rows leave no room on a CU beside them (LDS), so that the suffixes would come after them, one workgroup
  // a CU.  Many short suffixes are attended to by the launch that joins the partials instead, three workgroups a CU: (batch x heads
  // x group, prefix, suffix) 64 x 8 x 8, 32768, 256 of e4m3 114 -> 108 us; 64 x 8 x 8, 4096, 1000 64 -> 55; 33 x 16 x 4, 4096, 33 of
  // int8 35 -> 28; 32 x 8 x 8, 16384, 256 49 -> 47.  Fewer workgroups or longer suffixes lose: 64 x 2 x 8, 16384, 1000 41 -> 47;
  // 32 x 8 x 8, 8192, 4000 89 -> 99; so do the smaller blocks: 16 x 8 x 4, 32768, 500 42 -> 45.
  p.join_own = p.row_tiles == 16 && a->suffix.rows && a->suffix.rows <= 1024 && heads * batch >= 256;
  if (a->suffix.rows) cut(a->suffix.rows, p.join_own ? 1 : 256 / (heads * batch), TKA_MAX_SPLITS / 2, &p.own_splits, &p.own_tps);
  return p;
}

// The launches: a workgroup of up to 512 threads per item, then one of 256 per query row.
int launches_ok(int64_t batch, int64_t heads, int group, const Plan& p) {
  const int64_t segs = batch * heads, rows = segs * group;
  if (rows * p.parts() > kMaxItems || rows > kMaxThreads / 256) return TKA_EUNSUPPORTED;
  const int64_t items = p.row_tiles ? p.row_blocks * heads * p.shared_splits + segs * p.own_splits : segs;   // (at least those of each launch)
  return items <= kMaxThreads / 512 ? TKA_OK : TKA_EUNSUPPORTED;
}

int check_decode(const tka_kvq_flash_decode_args* a) {
  if (!a) return TKA_EINVAL;
  const tka_kv_cache& c = a->cache;
  int rc = check_cache(c, true, false);
  if (rc != TKA_OK) return rc;
  rc = check_row_stride(c);
  if (rc != TKA_OK) return rc;
  rc = check_query(a->q, a->dtype, a->group, a->q_stride_b, c.batch, c.num_kv_heads);
  if (rc != TKA_OK) return rc;
  rc = check_out(a->out, a->out_dtype, a->out_stride_b, c.batch, c.num_kv_heads, a->group);
  if (rc != TKA_OK) return rc;
  if (a->num_splits < 0 || a->num_splits > TKA_MAX_SPLITS) return TKA_EINVAL;
  if (a->idx_len > kMaxRows) return TKA_EUNSUPPORTED;
  if (a->kv_idx ? a->idx_len < 1 : (a->kv_count != nullptr || a->idx_len != 0)) return TKA_EINVAL;
  return launches_ok(c.batch, c.num_kv_heads, a->group, plan_decode(a));
}

int check_prefix(const tka_prefix_decode_args* a) {
  if (!a) return TKA_EINVAL;
  tka_kv_cache pre = a->prefix, suf = a->suffix;
  if (pre.format != suf.format || pre.num_kv_heads != suf.num_kv_heads || pre.batch != 1) return TKA_EINVAL;
  if (pre.rows < 0 || suf.rows < 0 || a->reserved0 != 0) return TKA_EINVAL;
  if (pre.rows + suf.rows == 0) return TKA_EINVAL;
  int rc;
  if (pre.rows && (rc = check_cache(pre, true, true)) != TKA_OK) return rc;
  if (suf.rows && (rc = check_cache(suf, true, true)) != TKA_OK) return rc;
  if ((pre.rows && (rc = check_row_stride(pre)) != TKA_OK) || (suf.rows && (rc = check_row_stride(suf)) != TKA_OK)) return rc;
  if (suf.batch < 1) return TKA_EINVAL;
  if (suf.batch > 65535) return TKA_EUNSUPPORTED;
  rc = check_query(a->q, a->dtype, a->group, a->q_stride_b, suf.batch, suf.num_kv_heads);
  if (rc != TKA_OK) return rc;
  rc = check_out(a->out, a->out_dtype, a->out_stride_b, suf.batch, suf.num_kv_heads, a->group);
  if (rc != TKA_OK) return rc;
  if (a->num_splits < 0 || a->num_splits > TKA_MAX_SPLITS / 2) return TKA_EINVAL;
  return launches_ok(suf.batch, suf.num_kv_heads, a->group, plan_prefix(a));
}

// The workspace: references and sums, then accumulators (nothing where one workgroup writes the result).
size_t partial_bytes(int64_t segs, int group, const Plan& p) {
  const size_t parts = p.to_workspace() ? (size_t)segs * group * (size_t)p.parts() : 0;
  return align_up(parts * 2 * sizeof(float), 256) + align_up(parts * TKA_HEAD_DIM * sizeof(float), 256) + 256;   // (never 0, which stands for a refused call)
}

int run_attend(KvAttendParams p, const Plan& plan, int dtype, int format, void* workspace, hipStream_t stream) {
  p.row_blocks = plan.row_blocks;
  p.shared_splits = plan.shared_splits;
  p.shared_tps = plan.shared_tps;
  p.own_splits = plan.join_own ? 0 : plan.own_splits;
  p.own_tps = plan.own_tps;
  p.num_splits = plan.parts();
  p.to_workspace = plan.to_workspace();
  const size_t parts = (size_t)p.batch * p.num_kv_heads * ((size_t)p.num_splits << p.group_log2);
  p.part_ml = (f32x2*)workspace;
  p.part_acc = (float*)((unsigned char*)workspace + align_up(parts * 2 * sizeof(float), 256));
  const int rc = launch_kv_attend(p, dtype, format, plan.row_tiles, stream);
  if (rc != TKA_OK || !p.to_workspace) return rc;
  return plan.join_own ? launch_kv_attend_join(p, dtype, format, stream) : launch_kv_combine(p, stream);
}

}  // namespace
}  // namespace tka

using namespace tka;

extern "C" {

int tka_kvq_write(const tka_kvq_write_args* a) {
  const int rc = check_copy(a, true);
  if (rc != TKA_OK) return rc;
  return launch_kvq_write(copy_params(a), a->dtype, a->cache.format, (hipStream_t)a->stream);
}

int tka_kvq_read(const tka_kvq_read_args* a) {
  const int rc = check_copy(a, false);
  if (rc != TKA_OK) return rc;
  return launch_kvq_read(copy_params(a), a->dtype, a->cache.format, (hipStream_t)a->stream);
}

int tka_kvq_scores(const tka_kvq_scores_args* a) {
  const int rc = check_scores(a);
  if (rc != TKA_OK) return rc;
  KvqScoresParams p;
  p.cache = rows_of(a->cache);
  p.q = a->q;
  p.q_stride_b = a->q_stride_b;
  p.kv_len = a->kv_len;
  p.scores = a->out_scores;
  p.batch = a->cache.batch;
  p.num_kv_heads = a->cache.num_kv_heads;
  p.group = a->group;
  p.scale = a->scale;
  return launch_kvq_scores(p, a->dtype, a->cache.format, (hipStream_t)a->stream);
}

size_t tka_kvq_flash_decode_workspace_bytes(const tka_kvq_flash_decode_args* a) {
  if (check_decode(a) != TKA_OK) return 0;
  const int64_t segs = (int64_t)a->cache.batch * a->cache.num_kv_heads;
  return partial_bytes(segs, a->group, plan_decode(a));
}

int tka_kvq_flash_decode(const tka_kvq_flash_decode_args* a) {
  const int rc = check_decode(a);
  if (rc != TKA_OK) return rc;
  if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < tka_kvq_flash_decode_workspace_bytes(a)) return TKA_EWORKSPACE;
  KvAttendParams p;
  memset(&p, 0, sizeof p);
  p.q = a->q;
  p.q_stride_b = a->q_stride_b;
  p.batch = a->cache.batch;
  p.num_kv_heads = a->cache.num_kv_heads;
  p.group_log2 = log2_of(a->group);
  p.own = rows_of(a->cache);
  p.own_len = a->kv_len;
  p.kv_idx = a->kv_idx;
  p.kv_count = a->kv_count;
  p.idx_len = a->idx_len;
  p.out = a->out;
  p.out_lse = a->out_lse;
  p.out_stride_b = a->out_stride_b;
  p.out_dtype = a->out_dtype;
  p.scale_log2e = a->scale * 1.44269504088896340736f;
  return run_attend(p, plan_decode(a), a->dtype, a->cache.format, a->workspace, (hipStream_t)a->stream);
}

size_t tka_prefix_decode_workspace_bytes(const tka_prefix_decode_args* a) {
  if (check_prefix(a) != TKA_OK) return 0;
  const int64_t segs = (int64_t)a->suffix.batch * a->suffix.num_kv_heads;
  return partial_bytes(segs, a->group, plan_prefix(a));
}

int tka_prefix_decode(const tka_prefix_decode_args* a) {
  const int rc = check_prefix(a);
  if (rc != TKA_OK) return rc;
  if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < tka_prefix_decode_workspace_bytes(a)) return TKA_EWORKSPACE;
  KvAttendParams p;
  memset(&p, 0, sizeof p);
  p.q = a->q;
  p.q_stride_b = a->q_stride_b;
  p.batch = a->suffix.batch;
  p.num_kv_heads = a->suffix.num_kv_heads;
  p.group_log2 = log2_of(a->group);
  if (a->prefix.rows) p.shared = rows_of(a->prefix);
  if (a->suffix.rows) p.own = rows_of(a->suffix);
  p.own_len = a->suffix_len;
  p.out = a->out;
  p.out_lse = a->out_lse;
  p.out_stride_b = a->out_stride_b;
  p.out_dtype = a->out_dtype;
  p.scale_log2e = a->scale * 1.44269504088896340736f;
  return run_attend(p, plan_prefix(a), a->dtype, a->prefix.format, a->workspace, (hipStream_t)a->stream);
}

int tka_kvq_test_row_tiles(int32_t row_tiles) {
  if (row_tiles != 0 && row_tiles != 1 && row_tiles != 2 && row_tiles != 4 && row_tiles != 8 && row_tiles != 16) return TKA_EINVAL;
  g_row_tiles.store(row_tiles, std::memory_order_relaxed);
  return TKA_OK;
}

}  // extern "C"
