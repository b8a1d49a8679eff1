// Quantising a K/V cache as it is written, reading it back, and the stage-1 scores over 8-bit keys.
//
//   kvq_write_kernel    A = max |x| of a row over 8 lanes of 16 elements each, then codes and scale (topk_attn_kvq.h)
//   kvq_read_kernel     code * scale, rounded to 16 bits
//   kvq_scores_kernel   the canonical 16-part dot product of topk_attn.h with codes as keys, times the row's scale
//
// All three are bound by the bytes they move: 256 + 132 per row and direction, 132 + 4 per scored row; short calls by the launch (3.8 to
// 4.3 us from call to call).  Measured: 3 prompts of up to 16385 tokens, 8 heads, fp16 to int8, 254 MB: 49 us, 5.2 TB/s; 2 x 32768 tokens
// back from int8 to bf16, 356 MB: 63 to 72 us, 5.0 to 5.7 TB/s; scores of 4 x 8 x 131072 rows of e4m3, 467 MB at lengths from half
// of it to all: 74 us, 6.3 TB/s.  (A copy of 4 GiB reads and writes 4.6 TB/s here, a kernel that only reads 7.1.)
#include <type_traits>

#include "kernels.hpp"
#include "kvq.hpp"

namespace tka {

namespace {

constexpr int kThreads = 256;
constexpr int kRowLanes = 8;                       // lanes of a row, 16 elements each
static_assert(kCopyRows == kThreads / kRowLanes, "");

// Code pairs / quads of one dword as fp32 numbers.
template <int FMT>
struct Codes;
template <>
struct Codes<TKA_KV_E4M3> {
  static __device__ __forceinline__ void widen(uint32_t w, float (&f)[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = lo[0];
    f[1] = lo[1];
    f[2] = hi[0];
    f[3] = hi[1];
  }
  // Smallest power of two s >= 2^-126 with top <= 448 s.  448 = 1.75 * 2^8: the exponent of `top` less 8, one more
  // where its significand exceeds 1.75.
  static __device__ __forceinline__ void scales(float top, float* scale, float* inverse) {
    const uint32_t u = __builtin_bit_cast(uint32_t, top);
    int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < 1 ? 1 : e;
    *scale = __builtin_bit_cast(float, (uint32_t)e << 23);
    *inverse = __builtin_bit_cast(float, (uint32_t)(254 - e) << 23);
  }
  static __device__ __forceinline__ uint32_t narrow(const float (&x)[4], float inverse) {   // x * inverse is exact, at most 448
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inverse, x[1] * inverse, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inverse, x[3] * inverse, w, true);
  }
};
template <>
struct Codes<TKA_KV_INT8> {
  static __device__ __forceinline__ void widen(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
  static __device__ __forceinline__ void scales(float top, float* scale, float* inverse) {
    const float least = __builtin_bit_cast(float, 1u << 23), most = __builtin_bit_cast(float, 253u << 23);   // 2^-126, 2^126
    *scale = fmaxf(__fdiv_rn(top, 127.0f), least);
    *inverse = top > 0.0f ? fminf(__fdiv_rn(127.0f, top), most) : most;
  }
  // The product is rounded to fp32 by itself (no fused multiply-add into the next step), then to a whole number.
  static __device__ __forceinline__ uint32_t narrow(const float (&x)[4], float inverse) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)__builtin_rintf(__fmul_rn(x[i], inverse)) & 0xffu) << (8 * i);
    return w;
  }
};

// A row is eight lanes: its maximum stays in three DPP steps, a wave stores eight rows of codes of one head, 1 KB without gaps where the
// cache lies head by head.  Row of this lane group and the lane's place in it.  Tokens go fastest: 2^tile_log2 of them (32 on long calls) lie next
// to each other in the scales of a head, a whole line of them.
struct CopyItem {
  bool there;
  int b, h;
  int64_t token, target;   // row of the 16-bit side, row of the cache
};
__device__ __forceinline__ CopyItem copy_item(const KvqCopyParams& p, uint32_t token_tiles) {
  const uint32_t row = threadIdx.x / kRowLanes;
  const uint32_t tile = blockIdx.x % token_tiles, pair0 = blockIdx.x / token_tiles;
  const uint32_t pair = (pair0 << (5 - p.tile_log2)) + (row >> p.tile_log2);
  CopyItem it;
  it.token = ((int64_t)tile << p.tile_log2) + (row & ((1u << p.tile_log2) - 1u));
  it.b = (int)(pair / (uint32_t)p.num_kv_heads);
  it.h = (int)(pair % (uint32_t)p.num_kv_heads);
  it.there = it.b < p.batch && it.token < p.num_tokens;
  it.target = it.token;
  if (it.there) {
    if (p.count) it.there = it.token < p.count[it.b];
    if (p.start) it.target += p.start[it.b];
    it.there = it.there && it.target >= 0 && it.target < p.cache.rows;
  }
  return it;
}

// max |x| of 16 elements as a 15-bit pattern: patterns of one sign order like their values, infinities and NaNs on top
__device__ __forceinline__ uint32_t top_pattern(const u32x4& a, const u32x4& b) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = a[i] & 0x7fff7fffu, y = b[i] & 0x7fff7fffu;
    m = max(m, max(max(x & 0xffffu, x >> 16), max(y & 0xffffu, y >> 16)));
  }
  m = max(m, dpp_u32<0xB1>(m));    // quad_perm [1,0,3,2]
  m = max(m, dpp_u32<0x4E>(m));    // quad_perm [2,3,0,1]
  m = max(m, dpp_u32<0x141>(m));   // row_half_mirror: the other quad of the eight lanes
  return m;
}

template <int DT, int FMT>
__device__ __forceinline__ u32x4 quantise16(const u32x4& a, const u32x4& b, float* scale) {
  const uint32_t top = top_pattern(a, b);
  const bool finite = top < (DT == TKA_F16 ? 0x7c00u : 0x7f80u);
  float inverse;
  Codes<FMT>::scales(Elem<DT>::widen((uint16_t)top), scale, &inverse);
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = Elem<DT>::get(i < 2 ? a : b, 4 * (i & 1) + e);
    w[i] = Codes<FMT>::narrow(x, inverse);
  }
  if (!finite) {
    *scale = __builtin_bit_cast(float, 0x7fc00000u);
    w = (u32x4){0u, 0u, 0u, 0u};
  }
  return w;
}

template <int DT, int FMT>
__global__ __launch_bounds__(kThreads) void kvq_write_kernel(KvqCopyParams p, uint32_t token_tiles) {
  const CopyItem it = copy_item(p, token_tiles);
  if (!it.there) return;   // (whole lane groups: the exchanges of the others stay inside their eight lanes)
  const int lane = threadIdx.x % kRowLanes;
  const int64_t in = it.b * p.stride_b + it.token * p.stride_n + it.h * p.stride_h + 32 * lane;
  const int64_t to = it.b * p.cache.stride_b + it.target * p.cache.stride_n + it.h * p.cache.stride_h + 16 * lane;
  const int64_t st = it.b * p.cache.scale_b + it.target * p.cache.scale_n + it.h * p.cache.scale_h;
  const u32x4 ka = __builtin_nontemporal_load((const u32x4*)(p.k + in)), kb = __builtin_nontemporal_load((const u32x4*)(p.k + in + 16));
  const u32x4 va = __builtin_nontemporal_load((const u32x4*)(p.v + in)), vb = __builtin_nontemporal_load((const u32x4*)(p.v + in + 16));
  float scale;
  __builtin_nontemporal_store((quantise16<DT, FMT>(ka, kb, &scale)), (u32x4*)((unsigned char*)p.cache.k + to));
  if (lane == 0) ((float*)p.cache.ks)[st] = scale;
  __builtin_nontemporal_store((quantise16<DT, FMT>(va, vb, &scale)), (u32x4*)((unsigned char*)p.cache.v + to));
  if (lane == 0) ((float*)p.cache.vs)[st] = scale;
}

// A finite number beyond the type's range becomes its largest (65504 is held as 256 * 2^8 in e4m3: half a step up); NaN stays.
template <int DT>
__device__ __forceinline__ uint16_t narrow_finite(float x) {
  const float most = DT == TKA_F16 ? 65504.0f : 3.3895313892515355e38f;
  const float y = fminf(fmaxf(x, -most), most);
  return Elem<DT>::narrow(x != x ? x : y);
}

template <int DT, int FMT>
__device__ __forceinline__ u32x4 dequantise8(const u32x2& w, float scale) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[4];
    Codes<FMT>::widen(w[i], f);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      o[2 * i + e] = (uint32_t)narrow_finite<DT>(f[2 * e] * scale) | ((uint32_t)narrow_finite<DT>(f[2 * e + 1] * scale) << 16);
  }
  return o;
}

template <int DT, int FMT>
__global__ __launch_bounds__(kThreads) void kvq_read_kernel(KvqCopyParams p, uint32_t token_tiles) {
  const CopyItem it = copy_item(p, token_tiles);
  if (!it.there) return;
  const int lane = threadIdx.x % kRowLanes;
  // a lane takes eight codes of either half of the row: a store then covers half a row without gaps, which is what the
  // streaming hint needs (with sixteen neighbouring codes a lane: 112 us instead of 84)
  const int64_t to = it.b * p.stride_b + it.token * p.stride_n + it.h * p.stride_h + 16 * lane;
  const int64_t at = it.b * p.cache.stride_b + it.target * p.cache.stride_n + it.h * p.cache.stride_h + 8 * lane;
  const int64_t st = it.b * p.cache.scale_b + it.target * p.cache.scale_n + it.h * p.cache.scale_h;
  const u32x2 ka = *(const u32x2*)(p.cache.k + at), kb = *(const u32x2*)(p.cache.k + at + 64);
  const u32x2 va = *(const u32x2*)(p.cache.v + at), vb = *(const u32x2*)(p.cache.v + at + 64);
  const float ks = p.cache.ks[st], vs = p.cache.vs[st];
  __builtin_nontemporal_store((dequantise8<DT, FMT>(ka, ks)), (u32x4*)(p.k + to));
  __builtin_nontemporal_store((dequantise8<DT, FMT>(kb, ks)), (u32x4*)(p.k + to + 128));
  __builtin_nontemporal_store((dequantise8<DT, FMT>(va, vs)), (u32x4*)(p.v + to));
  __builtin_nontemporal_store((dequantise8<DT, FMT>(vb, vs)), (u32x4*)(p.v + to + 128));
}

// A wave scores 64 tokens of a head: eight lanes a row, row u of group g is token 8g + u, so that lane 8g + x ends with the
// score of token 8g + x and scores and scales move in whole lines.  A lane holds two neighbouring parts (2i, 2i + 1) of the
// canonical sixteen; the butterfly runs over the lanes for the part distances 8, 4, 2 and ends inside the lane with 1.  Lane x
// takes the pair i = x (x < 4) or 11 - x, so that distance 8 is the DPP half mirror (i(7 - x) = i(x) ^ 4) and 4 and 2 are quad
// permutations: no exchange goes through the LDS crossbar, and the sums pair up as in the definition.
constexpr int kScoreRound = 64;
static_assert(kScoreTokens == (kThreads / kWave) * kScoreRound, "");

__device__ __forceinline__ float sum8(float p) {   // over eight lanes; every lane ends with the sum
  p = p + dpp_f32<0x141>(p);   // row_half_mirror
  p = p + dpp_f32<0x4E>(p);    // quad_perm [2,3,0,1]
  p = p + dpp_f32<0xB1>(p);    // quad_perm [1,0,3,2]
  return p;
}

template <int DT, int FMT>
__global__ __launch_bounds__(kThreads) void kvq_scores_kernel(KvqScoresParams p, uint32_t token_tiles) {
  const uint32_t seg = blockIdx.x / token_tiles, tile = blockIdx.x % token_tiles;
  const int b = (int)(seg / (uint32_t)p.num_kv_heads), h = (int)(seg % (uint32_t)p.num_kv_heads);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int g = lane >> 3, x = lane & 7;
  const int i = x < 4 ? x : 11 - x;
  int64_t len = p.cache.rows;
  if (p.kv_len) {
    const int64_t n = p.kv_len[b];
    len = n < 0 ? 0 : (n < len ? n : len);
  }
  // The rows are asked for before anything else; the sum of the group's queries (ascending, as in the definition) is made once
  // for the workgroup while they are on their way.
  const int64_t first = ((int64_t)tile * (kThreads / kWave) + wave) * kScoreRound, mine = first + lane;
  const int64_t last = len > 0 ? len - 1 : 0;
  const unsigned char* k = p.cache.k + b * p.cache.stride_b + h * p.cache.stride_h + 16 * i;
  const float* scales = p.cache.ks + b * p.cache.scale_b + h * p.cache.scale_h;
  u32x4 w[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) w[u] = __builtin_nontemporal_load((const u32x4*)(k + min(first + 8 * g + u, last) * p.cache.stride_n));
  const float ks = scales[min(mine, last) * p.cache.scale_n];
  __shared__ __align__(16) float sh_q[kHeadDim];
  if (threadIdx.x < kHeadDim) {
    const uint16_t* q = (const uint16_t*)p.q + (int64_t)b * p.q_stride_b + (int64_t)h * p.group * kHeadDim + threadIdx.x;
    uint16_t part[TKA_MAX_GROUP];
#pragma unroll
    for (int x = 0; x < TKA_MAX_GROUP; ++x) part[x] = q[(x < p.group ? x : 0) * kHeadDim];
    float sum = Elem<DT>::widen(part[0]);
#pragma unroll
    for (int x = 1; x < TKA_MAX_GROUP; ++x)
      if (x < p.group) sum += Elem<DT>::widen(part[x]);
    sh_q[threadIdx.x] = sum;
  }
  __syncthreads();
  float qf[16];
#pragma unroll
  for (int d = 0; d < 4; ++d) *(f32x4*)&qf[4 * d] = *(const f32x4*)&sh_q[16 * i + 4 * d];
  float dot = 0.0f;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    asm("" : "+v"(w[u]));   // (one row after the other: the compiler otherwise takes the bytes of all of them apart first)
    float part[2] = {0.0f, 0.0f}, f[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      Codes<FMT>::widen(w[u][d], f);
#pragma unroll
      for (int e = 0; e < 4; ++e) part[d >> 1] = __builtin_fmaf(qf[4 * d + e], f[e], part[d >> 1]);
    }
    const float s = sum8(part[0]) + sum8(part[1]);
    dot = x == u ? s : dot;
  }
  if (mine < p.cache.rows) p.scores[(int64_t)seg * p.cache.rows + mine] = mine < len ? (dot * ks) * p.scale : -INFINITY;
}

template <typename Launch>
int by_type(int dtype, int format, Launch launch) {
  if (dtype == TKA_F16) return format == TKA_KV_E4M3 ? launch(std::integral_constant<int, TKA_F16>(), std::integral_constant<int, TKA_KV_E4M3>())
                                                     : launch(std::integral_constant<int, TKA_F16>(), std::integral_constant<int, TKA_KV_INT8>());
  return format == TKA_KV_E4M3 ? launch(std::integral_constant<int, TKA_BF16>(), std::integral_constant<int, TKA_KV_E4M3>())
                               : launch(std::integral_constant<int, TKA_BF16>(), std::integral_constant<int, TKA_KV_INT8>());
}

}  // namespace

int launch_kvq_write(const KvqCopyParams& p0, int dtype, int format, hipStream_t stream) {
  KvqCopyParams p = p0;
  const CopyGrid grid = copy_grid((int64_t)p.batch * p.num_kv_heads, p.num_tokens);
  p.tile_log2 = grid.tile_log2;
  LaunchTimer timer("kvq_write", stream);
  return by_type(dtype, format, [&](auto dt, auto fmt) {
    kvq_write_kernel<dt(), fmt()><<<(uint32_t)grid.workgroups, kThreads, 0, stream>>>(p, (uint32_t)grid.token_tiles);
    return hip_status(hipGetLastError());
  });
}

int launch_kvq_read(const KvqCopyParams& p0, int dtype, int format, hipStream_t stream) {
  KvqCopyParams p = p0;
  const CopyGrid grid = copy_grid((int64_t)p.batch * p.num_kv_heads, p.num_tokens);
  p.tile_log2 = grid.tile_log2;
  LaunchTimer timer("kvq_read", stream);
  return by_type(dtype, format, [&](auto dt, auto fmt) {
    kvq_read_kernel<dt(), fmt()><<<(uint32_t)grid.workgroups, kThreads, 0, stream>>>(p, (uint32_t)grid.token_tiles);
    return hip_status(hipGetLastError());
  });
}

int launch_kvq_scores(const KvqScoresParams& p, int dtype, int format, hipStream_t stream) {
  const uint32_t tiles = (uint32_t)((p.cache.rows + kScoreTokens - 1) / kScoreTokens);
  const uint32_t grid = tiles * (uint32_t)p.batch * (uint32_t)p.num_kv_heads;
  LaunchTimer timer("kvq_scores", stream);
  return by_type(dtype, format, [&](auto dt, auto fmt) {
    kvq_scores_kernel<dt(), fmt()><<<grid, kThreads, 0, stream>>>(p, tiles);
    return hip_status(hipGetLastError());
  });
}

}  // namespace tka
