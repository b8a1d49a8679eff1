// Decode attention over 8-bit caches (dense or by token lists) and over a prefix that a batch shares with a suffix for each
// sequence, on the matrix cores (v_mfma_f32_16x16x32, fp32 accumulation).
//
//   S^T = K Q^T      A = K rows of 16 tokens (lane n + 16 j: token n, eight dims of quarter j per k-block), B = Q^T;
//                    lane (query row n, quarter j) gets the logits of tokens 4j .. 4j+3 of each 16;
//   softmax          one pass in the exp2 domain, running maximum and sum per query row, tokens spread over the quarters;
//   O^T = V^T P^T    B = P^T straight from the score registers: contraction slot (j, s) means token 4j + s (s < 4) or
//                    16 + 4j + s - 4 of a 32-token tile; A = V^T, loaded as rows (lane: dims 8n .. 8n+7 of the quarter's
//                    eight tokens) and transposed inside the lane with byte permutes.  Query rows stay in the lanes they
//                    have in S^T, so the running maximum rescales the accumulators without any exchange; accumulator
//                    (c, i) of lane (n, j) is O[query n][dim 32j + 8i + c].
//
// 8-bit rows: a code is exact as a 16-bit number, so K codes go to the type of q and V codes to fp16; the scale of a key
// row multiplies its logits, that of a value row its weight, both in fp32.  Weights enter the second product as fp16:
// 2^(x - m) * (scale / cap) * 2^9, with cap a power of two no scale seen so far exceeds (up to 2^127; accumulators move with it) and m a
// reference that no logit x exceeds by more than 6: at most 2^15, rounded by 2^-11 of themselves down to 2^-14 and by 2^-25
// below.  Where q is fp16 the remainder goes through the matrix cores as a second operand, so that the weights are as
// exact as the output.  16-bit rows: fp16 weights are held the same way without a cap; bf16 weights have fp32's range but
// 8 bits only, their remainder always is a second operand, and they are held times 2^-32, so that no sum of the largest
// numbers overflows.  (The factor sits in the exponent, and the sum of the weights has it too.)
//
// The reference m of a row only moves when weights have grown by 2^6: after the first tiles that is rare, and a tile then
// needs neither the row's maximum, an exchange between lanes, nor a pass over the accumulators.
//
// Results of waves and splits are joined normalised, out = sum (l_s 2^(m_s - M) / L) o_s: they stay in the range of V.
//
// A workgroup is one (source, batch entry or block of query rows, head, split); its waves take 32-token tiles in turn and
// are joined in LDS, the splits by a second launch.  The shared source multiplies a block of query rows (entries x group) with each
// K / V tile.
//
// What bounds it: the bytes of the cache for a decode (4 x 8 x 32768 rows of e4m3, lengths from half of it to all, 225 MB: 44 us,
// 5.1 TB/s); two launches of about 4 us each for a short call; the latency of the gather for a list (8 x 8 lists of up to 2128 of 32768
// rows of int8, three quarters full: 15.3 us, 11.8 of them in the first launch, which fetches 39 MB of lines, 3.3 TB/s; 384 workgroups, some
// of them without rows, are one or two waves a SIMD with three rounds of dependent loads each; e4m3 15.0); the bytes, then the issue of the products,
// for a prefix (16 x 8 x 4 query rows over 32768 + 500 rows of 16 bits, 159 MB: 41 us, 3.9 TB/s; larger blocks of query rows: at
// kv_attend_wide_kernel).  Splits are cut for the capacity of a cache, not for the lengths it holds: 4 x 8 heads that hold 16384 tokens
// take 26.5 us in a cache of 16384 and 118 in one of 131072, where most workgroups have no rows (4096 tokens: 12.6 and 64).
//
// Joining the splits in the launch itself, by the last workgroup of a row, took longer than the second launch does (8 splits of one
// head 8.7 us against 8.1, 32 heads 29.7 against 11.5: the XCDs have no L2 in common, so that flags and partials go through memory).
#include <type_traits>

#include "kernels.hpp"
#include "kvq.hpp"

namespace tka {

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kTile = kAttendTile;
constexpr float kNoReference = -3.402823466e38f;   // of a row that has seen no key: what lies above it moves it
constexpr int kStagedIds = 2048;
constexpr int kLdsRow = kHeadDim + 4;   // (rows 4 floats apart in the banks)

__device__ __forceinline__ f32x4 mfma_f16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_bf16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (F16) return mfma_f16(a, b, c);
  else return mfma_bf16(a, b, c);
}
// (by value: __builtin_bit_cast of an element of a vector takes the vector's first element, whichever was named)
__device__ __forceinline__ f16x2 as_f16(uint32_t x) { return __builtin_bit_cast(f16x2, x); }
__device__ __forceinline__ uint32_t as_bits(f16x2 x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const f16x2 v = {(_Float16)lo, (_Float16)hi};
  return as_bits(v);
}
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}

// Two codes (bytes 2 HI and 2 HI + 1 of w) as a pair of 16-bit numbers, exactly.
template <int FMT, bool F16, int HI>
__device__ __forceinline__ uint32_t widen_pair(uint32_t w) {
  if constexpr (FMT == TKA_KV_E4M3) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI != 0));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI != 0));
  } else if constexpr (F16) {
    // (w has its bytes offset by 128 already) 0x6400 | u is the fp16 number 1024 + u
    const uint32_t biased = __builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u);
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, biased) - off);
  } else {
    const float lo = (float)(int8_t)(w >> (16 * HI)), hi = (float)(int8_t)(w >> (16 * HI + 8));
    return pack_bf16(lo, hi);   // (whole numbers below 2^8: exact)
  }
}
// What widen_pair expects of a dword of codes.
template <int FMT, bool F16>
__device__ __forceinline__ uint32_t prepare_codes(uint32_t w) {
  if constexpr (FMT == TKA_KV_INT8 && F16) return w ^ 0x80808080u;
  else return w;
}

template <int FMT>
constexpr bool kQuantised = FMT != TKA_KV_16BIT;

// K registers of a 16-token tile (token n of the lane): 16-bit rows: k-block kb is dims 32 kb + 8 j .. + 7; 8-bit rows: a
// 16-byte load x covers dims 64 x + 16 j .. + 15, k-blocks 2x and 2x + 1 their halves.
template <int FMT>
struct KTile {
  static constexpr int kLoads = kQuantised<FMT> ? 2 : 4;
  u32x4 w[kLoads];
};
template <int FMT>
__device__ __forceinline__ int k_dim(int kb, int j) { return kQuantised<FMT> ? 64 * (kb >> 1) + 16 * j + 8 * (kb & 1) : 32 * kb + 8 * j; }

template <int FMT, bool F16>
__device__ __forceinline__ u32x4 k_frag(const KTile<FMT>& t, int kb) {
  if constexpr (!kQuantised<FMT>) {
    return t.w[kb];
  } else {
    const uint32_t a = prepare_codes<FMT, F16>(t.w[kb >> 1][2 * (kb & 1)]), b = prepare_codes<FMT, F16>(t.w[kb >> 1][2 * (kb & 1) + 1]);
    return (u32x4){widen_pair<FMT, F16, 0>(a), widen_pair<FMT, F16, 1>(a), widen_pair<FMT, F16, 0>(b), widen_pair<FMT, F16, 1>(b)};
  }
}

// V registers: dims 8n .. 8n+7 of the eight slot tokens.
template <int FMT>
using VRow = typename std::conditional<kQuantised<FMT>, u32x2, u32x4>::type;

// Rows that a loop carries along are to stay in the registers as they were loaded: the compiler otherwise carries the bytes that
// their conversion begins with, in a register each (int8 keys, bf16 queries: 64 registers more than there are).
template <int FMT>
__device__ __forceinline__ void hold(KTile<FMT> (&kt)[2], VRow<FMT> (&vr)[8]) {
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < KTile<FMT>::kLoads; ++y) asm("" : "+v"(kt[x].w[y]));
#pragma unroll
  for (int s = 0; s < 8; ++s) asm("" : "+v"(vr[s]));
}

// V^T operands of output dims c = 2 D and 2 D + 1 (of the lane's eight): element s = token of slot s.
template <int FMT, int D>
__device__ __forceinline__ void v_frags(const VRow<FMT> (&v)[8], u32x4* even, u32x4* odd) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (!kQuantised<FMT>) {
      (*even)[w] = __builtin_amdgcn_perm(v[2 * w + 1][D], v[2 * w][D], 0x05040100u);
      (*odd)[w] = __builtin_amdgcn_perm(v[2 * w + 1][D], v[2 * w][D], 0x07060302u);
    } else {
      // bytes: token 2w dim 2D, token 2w+1 dim 2D, then dim 2D + 1 of the two
      const uint32_t sel = (D & 1) ? 0x07030602u : 0x05010400u;
      const uint32_t pair = prepare_codes<FMT, true>(__builtin_amdgcn_perm(v[2 * w + 1][D >> 1], v[2 * w][D >> 1], sel));
      (*even)[w] = widen_pair<FMT, true, 0>(pair);
      (*odd)[w] = widen_pair<FMT, true, 1>(pair);
    }
  }
}

// token of contraction slot (quarter j, s) inside a 32-token tile
__device__ __forceinline__ int slot_token(int j, int s) { return s < 4 ? 4 * j + s : 16 + 4 * j + (s - 4); }

__device__ __forceinline__ float max_over_quarters(float x) {
  x = fmaxf(x, __builtin_bit_cast(float, lane_xor<16>(__builtin_bit_cast(uint32_t, x))));
  return fmaxf(x, __builtin_bit_cast(float, lane_xor<32>(__builtin_bit_cast(uint32_t, x))));
}
__device__ __forceinline__ float sum_over_quarters(float x) {
  x += __builtin_bit_cast(float, lane_xor<16>(__builtin_bit_cast(uint32_t, x)));
  return x + __builtin_bit_cast(float, lane_xor<32>(__builtin_bit_cast(uint32_t, x)));
}

constexpr int kJoined = 4;   // waves that are joined in one go
struct AttendLds {
  float acc[kJoined][16][kLdsRow];
  union {
    struct {
      float m[kJoined][16];
      float l[kJoined][16];
    };
    float state[kJoined][kWave][3];   // of more than four waves: reference, sum, cap
  };
};

template <bool F16>
constexpr float kWeightLog2 = F16 ? 9.0f : -32.0f;   // weights are held times 2^this
template <bool F16>
constexpr float kMostWeight = F16 ? 32704.0f : 0x1p-26f;   // 2^6 times that: the reference moves when eight weights add up to more
// (in fp16 a little less: a weight times a scale of just below twice the largest cap, 2^127, has to stay below 65504)

// Positions [begin, end) of the rows of one entry and head (of a token list where there is one).
struct AttendSource {
  const unsigned char* k;
  const unsigned char* v;
  const float* ks;
  const float* vs;
  int64_t stride_n, scale_n;
  const int32_t* idx;
  int len;                  // rows of the cache that listed ids may name
  int begin, end;           // (uniform over the wave, like everything here)
};

// What a workgroup attends to, one source after the other, for the query rows [row0, row0 + 16 RT) below row_end; query row
// r is head h * group + r % group of batch entry b0 + r / group.
struct AttendItem {
  AttendSource first, second;
  bool two;
  int b0, h, row0, row_end, slot;
};

// Dims d0 .. d0+7 of a finished row (query head hq of entry b) and, with the first of them, its lse.
__device__ __forceinline__ void store_row(const KvAttendParams& p, int b, int hq, int d0, const f32x4& lo, const f32x4& hi, float M, float L, float l_log2) {
  u32x4 o;
  if (p.out_dtype == TKA_F16) o = (u32x4){pack_f16(lo[0], lo[1]), pack_f16(lo[2], lo[3]), pack_f16(hi[0], hi[1]), pack_f16(hi[2], hi[3])};
  else o = (u32x4){pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]), pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3])};
  *(u32x4*)((uint16_t*)p.out + b * p.out_stride_b + (int64_t)hq * kHeadDim + d0) = o;
  if (p.out_lse && d0 == 0)
    p.out_lse[(((int64_t)b * p.num_kv_heads) << p.group_log2) + hq] = L > 0.0f || L != L ? (M + (__builtin_log2f(L) - l_log2)) * 0.69314718055994531f : -INFINITY;
}

// Twice the power of two at or above x (x >= 0), 2^-110 at least and 2^127 at most.
__device__ __forceinline__ float power_above(float x) {
  const uint32_t e = ((__builtin_bit_cast(uint32_t, x) + 0x7fffffu) & 0x7f800000u) + 0x800000u;
  return __builtin_bit_cast(float, min(max(e, 17u << 23), 0x7f000000u));
}
// 1 / x of a power of two from 2^-126 to 2^127 (whose reciprocal is a subnormal number).
__device__ __forceinline__ float power_inverse(float x) {
  return __builtin_bit_cast(float, max((254u << 23) - __builtin_bit_cast(uint32_t, x), 0x400000u));
}

// What lanes of the wave have stored to LDS is there for its other lanes to load (the LDS serves a wave's accesses in order: this
// holds the compiler to that order, and costs nothing).
__device__ __forceinline__ void wave_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The power of two at or above |x|, 2^-126 at least and 2^127 at most.
__device__ __forceinline__ float power_at(float x) {
  const uint32_t e = (min(__builtin_bit_cast(uint32_t, x) & 0x7fffffffu, 0x7f000000u) + 0x7fffffu) & 0x7f800000u;
  return __builtin_bit_cast(float, max(e, 1u << 23));
}

// What a wave holds of its 16 RT query rows (row n of each sixteen in the lanes n, n + 16, n + 32, n + 48).
template <int DT, int FMT, int RT>
struct Rows {
  static constexpr bool kQF16 = DT == TKA_F16;
  static constexpr bool kPF16 = kQuantised<FMT> || DT == TKA_F16;   // type of the second product
  static constexpr bool kSplit = !kPF16 || DT == TKA_F16;           // weights in two parts
  u32x4 q[RT][4];
  float m_ref[RT], l_run[RT];   // l_run: this quarter's share
  f32x4 acc[RT][8];
  float cap;

  // Rows [row0, row0 + 16 RT) below row_end; row r is head h * group + r % group of entry b0 + r / group.
  __device__ __forceinline__ void begin(const KvAttendParams& p, int b0, int h, int row0, int row_end) {
    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4, group = 1 << p.group_log2;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = row0 + 16 * r + n;
      const bool there = row < row_end;
      const int rr = there ? row : 0;
      const uint16_t* of = (const uint16_t*)p.q + (int64_t)(b0 + (rr >> p.group_log2)) * p.q_stride_b +
                           (int64_t)(h * group + (rr & (group - 1))) * kHeadDim;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        q[r][kb] = *(const u32x4*)(of + k_dim<FMT>(kb, j));
        if (!there) q[r][kb] = (u32x4){0u, 0u, 0u, 0u};
      }
      m_ref[r] = kNoReference;
      l_run[r] = 0.0f;
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[r][c] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    cap = __builtin_bit_cast(float, 17u << 23);   // 2^-110: the least cap (its reciprocal stays in range)
  }

  // The cap moves to `to`, a power of two, and the accumulators with it.
  __device__ __forceinline__ void raise_cap(float to) {
    const float drop = cap / to;
    cap = to;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[r][c] *= drop;
  }

  // Logits of a tile of 32 tokens, before their factors.  key_frag(x, kb): operand of sixteen x and k-block kb.
  template <typename KeyFrag>
  __device__ __forceinline__ void scores(f32x4 (&sc)[RT][2], KeyFrag key_frag) const {
#pragma unroll
    for (int r = 0; r < RT; ++r) sc[r][0] = sc[r][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const u32x4 a = key_frag(x, kb);
#pragma unroll
        for (int r = 0; r < RT; ++r) sc[r][x] = mfma<kQF16>(a, q[r][kb], sc[r][x]);
      }
  }

  // The rest of it.  kf: factors of the slot tokens' logits, vs: their value scales; masked: bit s = slot s has no row
  // (any_masked: some lane has one); value_frags(D, even, odd): operands of output dims 2 D and 2 D + 1.
  // tile_scale (SCALED): a power of two that the value operands have been divided by, with their scales in them (vs is then not
  // looked at); rest, where `uneven`: what the tile's scales have beside that, for the weights.
  template <bool SCALED, typename ValueFrags>
  __device__ __forceinline__ void attend(f32x4 (&sc)[RT][2], float (&kf)[8], float (&vs)[8], float tile_scale, bool uneven, const float* rest,
                                         uint32_t masked, bool any_masked, ValueFrags value_frags) {
    // masked slots have no weight (and their value rows are zeros: no 0 * inf, no 0 * NaN)
    if (any_masked) {
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (masked >> s & 1u) {
          vs[s] = 0.0f;
          kf[s] = 1.0f;
#pragma unroll
          for (int r = 0; r < RT; ++r) sc[r][s >> 2][s & 3] = -INFINITY;
        }
    }
    float weight[8];   // scale of a slot's value row over the cap
    float unit_log2 = kWeightLog2<kPF16>, back = 1.0f;   // log2 of the unit that the weights are held in; what takes their sum back to 2^kWeightLog2
    if constexpr (SCALED) {
      if (tile_scale > cap) raise_cap(tile_scale);
      const int below = max((int)(__builtin_bit_cast(uint32_t, tile_scale) >> 23) - (int)(__builtin_bit_cast(uint32_t, cap) >> 23), -40);   // (2^-40 of the cap: nothing)
      unit_log2 += (float)below;
      back = __builtin_bit_cast(float, (uint32_t)(127 - below) << 23);
    } else if constexpr (kQuantised<FMT>) {
      float top = fabsf(vs[0]);
#pragma unroll
      for (int s = 1; s < 8; ++s) top = fmaxf(top, fabsf(vs[s]));
      if (__ballot(top > cap) != 0ull) raise_cap(power_above(max_over_quarters(top)));
      const float unit = power_inverse(cap);
#pragma unroll
      for (int s = 0; s < 8; ++s) weight[s] = vs[s] * unit;
    }

    // ---- weights.  A lane's sum that exceeds the headroom (an infinite one in the first tile) sends the tile through the
    // pass that moves the references.
    u32x4 pf[RT], pf_lo[RT];
    float ps[RT][8], sum[RT], most = 0.0f;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int s = 0; s < 8; ++s) ps[r][s] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][s >> 2][s & 3], kf[s], unit_log2 - m_ref[r]));
      sum[r] = ((ps[r][0] + ps[r][1]) + (ps[r][2] + ps[r][3])) + ((ps[r][4] + ps[r][5]) + (ps[r][6] + ps[r][7]));
      most = fmaxf(most, sum[r]);
    }
    if (__ballot(most > kMostWeight<kPF16>) != 0ull) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float xs[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) xs[s] = sc[r][s >> 2][s & 3] * kf[s];
        float top = xs[0];
#pragma unroll
        for (int s = 1; s < 8; ++s) top = fmaxf(top, xs[s]);
        const float m_new = fmaxf(m_ref[r], max_over_quarters(top));
        const float alpha = __builtin_amdgcn_exp2f(m_ref[r] - m_new);
        m_ref[r] = m_new;
        l_run[r] *= alpha;
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[r][c] *= alpha;
#pragma unroll
        for (int s = 0; s < 8; ++s) ps[r][s] = __builtin_amdgcn_exp2f(xs[s] + (unit_log2 - m_new));
        sum[r] = ((ps[r][0] + ps[r][1]) + (ps[r][2] + ps[r][3])) + ((ps[r][4] + ps[r][5]) + (ps[r][6] + ps[r][7]));
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) l_run[r] = SCALED ? __builtin_fmaf(sum[r], back, l_run[r]) : l_run[r] + sum[r];
    if (SCALED && uneven) {
      const float* of = rest + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const f32x4 f = *(const f32x4*)(of + 16 * x);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) ps[r][4 * x + i] *= f[i];
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float a = ps[r][2 * w], b = ps[r][2 * w + 1];
        if constexpr (kPF16) {
          const float x = kQuantised<FMT> && !SCALED ? a * weight[2 * w] : a, y = kQuantised<FMT> && !SCALED ? b * weight[2 * w + 1] : b;
          pf[r][w] = pack_f16(x, y);
          if constexpr (kSplit) {
            const f16x2 h = as_f16(pf[r][w]);
            pf_lo[r][w] = pack_f16(x - (float)h[0], y - (float)h[1]);
          }
        } else {
          pf[r][w] = pack_bf16(a, b);
          pf_lo[r][w] = pack_bf16(a - __builtin_bit_cast(float, pf[r][w] << 16), b - __builtin_bit_cast(float, pf[r][w] & 0xffff0000u));
        }
      }
    }

    // ---- values
    const auto values = [&](auto d) {
      constexpr int D = decltype(d)::value;
      u32x4 even, odd;
      value_frags(d, &even, &odd);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        acc[r][2 * D] = mfma<kPF16>(even, pf[r], acc[r][2 * D]);
        acc[r][2 * D + 1] = mfma<kPF16>(odd, pf[r], acc[r][2 * D + 1]);
        if constexpr (kSplit) {
          acc[r][2 * D] = mfma<kPF16>(even, pf_lo[r], acc[r][2 * D]);
          acc[r][2 * D + 1] = mfma<kPF16>(odd, pf_lo[r], acc[r][2 * D + 1]);
        }
      }
    };
    values(std::integral_constant<int, 0>());
    values(std::integral_constant<int, 1>());
    values(std::integral_constant<int, 2>());
    values(std::integral_constant<int, 3>());
  }
};

// Rows of a dense source, a tile of 32 positions from `start`: key rows 16x + n, value and scale rows the slot tokens.  A scalar
// base and 32-bit lane offsets (32 strides fit, the host checks); rows that a source of less than 32 does not have are
// replaced by its last.
template <int FMT>
struct DenseTiles {
  uint32_t k_off[2], v_off[8];
  int last;
  bool vector_scales;

  __device__ __forceinline__ void begin(const AttendSource& it) {
    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const uint32_t stride = (uint32_t)it.stride_n;
    last = min(it.end, kTile) - 1;
    vector_scales = it.scale_n == 1 && it.end >= kTile;
#pragma unroll
    for (int x = 0; x < 2; ++x) k_off[x] = (uint32_t)min(16 * x + n, last) * stride + 16u * j;
#pragma unroll
    for (int s = 0; s < 8; ++s) v_off[s] = (uint32_t)min(slot_token(j, s), last) * stride + (kQuantised<FMT> ? 8u : 16u) * n;
  }
  __device__ __forceinline__ void scales(const AttendSource& it, const float* of_source, int start, float (&f)[8]) const {
    const int j = (threadIdx.x & 63) >> 4;
    const float* base = of_source + (int64_t)start * it.scale_n;
    if (vector_scales) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const f32x4u v = *(const f32x4u*)(base + 16 * x + 4u * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * x + i] = v[i];
      }
    } else {
      int most = last;
      asm("" : "+s"(most));   // (the eight offsets are made here, not kept in registers over the loop)
#pragma unroll
      for (int s = 0; s < 8; ++s) f[s] = *(const float*)((const unsigned char*)base + (uint32_t)min(slot_token(j, s), most) * (uint32_t)(4 * it.scale_n));
    }
  }
  __device__ __forceinline__ void keys(const AttendSource& it, int start, KTile<FMT> (&kt)[2], float (&ks)[8]) const {
    key_rows(it, start, kt);
    if constexpr (kQuantised<FMT>) scales(it, it.ks, start, ks);
  }
  __device__ __forceinline__ void values(const AttendSource& it, int start, VRow<FMT> (&vr)[8], float (&vs)[8]) const {
    value_rows<true>(it, start, vr);
    if constexpr (kQuantised<FMT>) scales(it, it.vs, start, vs);
  }
  __device__ __forceinline__ void key_rows(const AttendSource& it, int start, KTile<FMT> (&kt)[2]) const {
    const unsigned char* base = it.k + (int64_t)start * it.stride_n;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < KTile<FMT>::kLoads; ++y) kt[x].w[y] = *(const u32x4*)(base + k_off[x] + 64 * y);
  }
  // STREAM: with the hint that the rows are not read again (a request covers whole lines).  All but the blocks of 128 and 256 query
  // rows give it, also for rows that several workgroups read.  With and without it, us: decode of 4 x 8 x 32768 rows of e4m3 46.1 and 53.0;
  // prefixes of 32768 rows of 16 bits, 16 x 8 x 4 39.8 and 45.8, 32 x 8 x 4 47.1 and 50.2, 64 x 8 x 8 134 and 141; one-launch calls the
  // same; it loses for 8-bit rows that are shared: prefixes of e4m3, 16 x 8 x 4 32.3 and 29.8, 32 x 8 x 4 45.9 and 41.4, a decode of
  // 16 x 8 x 4 over one cache of 32768 110 and 106.
  template <bool STREAM>
  __device__ __forceinline__ void value_rows(const AttendSource& it, int start, VRow<FMT> (&vr)[8]) const {
    const unsigned char* base = it.v + (int64_t)start * it.stride_n;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const VRow<FMT>* row = (const VRow<FMT>*)(base + v_off[s]);
      vr[s] = STREAM ? __builtin_nontemporal_load(row) : *row;
    }
  }
};

// A dense tile that the end cuts starts earlier, at the last 32 rows that there are, and its first positions are masked.
__device__ __forceinline__ int tile_start(int tile, int end) { return end - tile >= kTile ? tile : max(end - kTile, 0); }
__device__ __forceinline__ uint32_t tile_mask(int start, int tile, int end) {
  const int j = (threadIdx.x & 63) >> 4;
  uint32_t masked = 0;
#pragma unroll
  for (int s = 0; s < 8; ++s) masked |= start + slot_token(j, s) < tile || start + slot_token(j, s) >= end ? 1u << s : 0u;
  return masked;
}
template <int FMT>
__device__ __forceinline__ void clear_masked(uint32_t masked, VRow<FMT> (&vr)[8]) {
#pragma unroll
  for (int s = 0; s < 8; ++s)
    if (masked >> s & 1u) vr[s] = VRow<FMT>{};
}

// Partial of one split (a join follows) or the finished row, dims d0 .. d0 + 7.
template <bool F16>
__device__ __forceinline__ void store_result(const KvAttendParams& p, int b, int hq, int slot, int d0, const f32x4& lo, const f32x4& hi, float M, float L) {
  if (p.to_workspace) {
    const int64_t at = ((((int64_t)b * p.num_kv_heads) << p.group_log2) + hq) * p.num_splits + slot;
    f32x4* to = (f32x4*)(p.part_acc + at * kHeadDim + d0);
    to[0] = lo;
    to[1] = hi;
    // (the sum as it is held belongs to a reference that much lower)
    if (d0 == 0) p.part_ml[at] = (f32x2){M == kNoReference ? M : M - kWeightLog2<F16>, L};
  } else {
    store_row(p, b, hq, d0, lo, hi, M, L, kWeightLog2<F16>);
  }
}

// Joins what 256 threads hold of a workgroup's own rows (thread: dims d0 .. d0+7 of query row `row`, reference M in base 2, sum L;
// part `part` of `parts` for each row) with the partials of the shared rows, and writes the rows.
__device__ __forceinline__ void join_shared(const KvAttendParams& p, int b, int hq, int d0, int slot, int part, int parts, f32x4 lo, f32x4 hi, float M,
                                            float L, float (&sh)[16][kLdsRow]) {
  const int S = p.num_splits, x = threadIdx.x & 15;
  const int64_t at = ((((int64_t)b * p.num_kv_heads) << p.group_log2) + hq) * S;
  const f32x2* ml = p.part_ml + at;
  const f32x4* pa = (const f32x4*)(p.part_acc + at * kHeadDim + d0);
  float top = M;
  for (int s = x; s < S; s += 16) top = fmaxf(top, ml[s][0]);
#pragma unroll
  for (int y = 8; y >= 1; y >>= 1) top = fmaxf(top, __shfl_xor(top, y, 64));
  float sum = 0.0f;
  for (int s = x; s < S; s += 16) sum += ml[s][1] * __builtin_amdgcn_exp2f(ml[s][0] - top);
#pragma unroll
  for (int y = 8; y >= 1; y >>= 1) sum += __shfl_xor(sum, y, 64);
  const float own = L * __builtin_amdgcn_exp2f(M - top);
  sum += own;
  const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
  lo *= part ? 0.0f : own * inv;
  hi *= part ? 0.0f : own * inv;
  for (int s0 = part; s0 < S; s0 += 4 * parts) {
    f32x4 a[4], c[4];
    float w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * parts < S ? s0 + u * parts : s0;
      a[u] = pa[(int64_t)s * (kHeadDim / 4)];
      c[u] = pa[(int64_t)s * (kHeadDim / 4) + 1];
      w[u] = ml[s][1] * __builtin_amdgcn_exp2f(ml[s][0] - top) * inv;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + u * parts < S) {
        lo += a[u] * w[u];
        hi += c[u] * w[u];
      }
  }
  __syncthreads();   // (the own rows have been read)
  *(f32x4*)&sh[slot][d0] = lo;
  *(f32x4*)&sh[slot][d0 + 4] = hi;
  __syncthreads();
  if (part) return;
  for (int y = 1; y < parts; ++y) {
    lo += *(const f32x4*)&sh[slot + (y << p.group_log2)][d0];
    hi += *(const f32x4*)&sh[slot + (y << p.group_log2)][d0 + 4];
  }
  store_row(p, b, hq, d0, lo, hi, top, sum, 0.0f);
}

// JOIN: the workgroup then joins its rows with the partials of the shared source and writes them.
template <int DT, int FMT, int RT, bool INDEXED, int WAVES, bool JOIN = false>
__device__ __forceinline__ void attend(const KvAttendParams& p, const AttendItem& item, AttendLds& sh, int32_t* sh_ids) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, j = lane >> 4;
  const int group = 1 << p.group_log2;
  Rows<DT, FMT, RT> rows;
  rows.begin(p, item.b0, item.h, item.row0, item.row_end);

  // One source: its tiles go round the waves, `turn` is this wave's first.  The keys of the next tile are asked for as soon as
  // those of this one are in the matrix cores, its values behind this tile's.
  const auto attend_source = [&](const AttendSource& it, int turn) {
    KTile<FMT> kt[2];
    VRow<FMT> vr[8];
    float ks[8], vs[8];
    DenseTiles<FMT> dense;
    if constexpr (!INDEXED) dense.begin(it);
    // Listed: rows by the ids of the positions in LDS, -1 replaced by row 0.
    const auto listed_scales = [&](const float* of_source, int start, float (&f)[8]) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const i32x4 id = *(const i32x4*)&sh_ids[start + 16 * x + 4 * j];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * x + i] = of_source[(int64_t)max(id[i], 0) * it.scale_n];
      }
    };
    const auto load_keys = [&](int start) {
      if constexpr (INDEXED) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const unsigned char* row = it.k + (int64_t)max(sh_ids[start + 16 * x + n], 0) * it.stride_n + 16 * j;
#pragma unroll
          for (int y = 0; y < KTile<FMT>::kLoads; ++y) kt[x].w[y] = *(const u32x4*)(row + 64 * y);
        }
        listed_scales(it.ks, start, ks);
      } else {
        dense.keys(it, start, kt, ks);
      }
    };
    const auto load_values = [&](int start) {
      if constexpr (INDEXED) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const i32x4 id = *(const i32x4*)&sh_ids[start + 16 * x + 4 * j];
#pragma unroll
          for (int i = 0; i < 4; ++i) vr[4 * x + i] = *(const VRow<FMT>*)(it.v + (int64_t)max(id[i], 0) * it.stride_n + (kQuantised<FMT> ? 8 : 16) * n);
        }
        listed_scales(it.vs, start, vs);
      } else {
        dense.values(it, start, vr, vs);
      }
    };

    // Positions [begin, end) (listed ones are filled up to whole tiles with -1).
    const auto run = [&](int begin, int end) {
      int rest = end - begin - turn * kTile;   // positions from this tile's first on
      if (rest <= 0) return;
      int tile = begin + turn * kTile;
      int start = INDEXED ? tile : tile_start(tile, end);
      load_keys(start);
      load_values(start);
      while (true) {
        asm("" : "+s"(start));   // (addresses are made from it in scalar registers, not carried along in vector registers)
        const bool more = rest > WAVES * kTile;
        const int next_tile = tile + WAVES * kTile;
        const int next = INDEXED || rest >= (WAVES + 1) * kTile ? next_tile : max(end - kTile, 0);
        uint32_t masked = 0;
        bool any_masked;
        if constexpr (INDEXED) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const i32x4 id = *(const i32x4*)&sh_ids[start + 16 * x + 4 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i) masked |= id[i] < 0 ? 1u << (4 * x + i) : 0u;
          }
          any_masked = __ballot(masked != 0) != 0ull;
        } else {
          any_masked = rest < kTile;
          if (any_masked) masked = tile_mask(start, tile, end);
        }
        float kf[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) kf[s] = kQuantised<FMT> ? ks[s] * p.scale_log2e : p.scale_log2e;
        f32x4 sc[RT][2];
        rows.scores(sc, [&](int x, int kb) { return k_frag<FMT, Rows<DT, FMT, RT>::kQF16>(kt[x], kb); });
        if (more) load_keys(next);
        if (any_masked) clear_masked<FMT>(masked, vr);
        rows.template attend<false>(sc, kf, vs, 0.0f, false, nullptr, masked, any_masked, [&](auto d, u32x4* even, u32x4* odd) { v_frags<FMT, decltype(d)::value>(vr, even, odd); });
        if (!more) break;
        load_values(next);
        tile = next_tile;
        start = next;
        rest -= WAVES * kTile;
      }
    };
    if constexpr (INDEXED) {   // the ids of up to kStagedIds positions at a time, skipped ones as -1
      for (int begin = it.begin, rest = it.end - it.begin; rest > 0; begin += kStagedIds, rest -= kStagedIds) {
        const int count = min(rest, kStagedIds);
        if (begin > it.begin) __syncthreads();
        for (int i = tid; i < (count + kTile - 1) / kTile * kTile; i += WAVES * kWave) {
          const int id = i < count ? it.idx[begin + i] : -1;
          sh_ids[i] = id >= 0 && id < it.len ? id : -1;
        }
        __syncthreads();
        run(0, count);
      }
    } else {
      run(it.begin, it.end);
    }

  };
  attend_source(item.first, wave);
  if (item.two) {   // the waves that had one tile less go on
    const int before = ((item.first.end - item.first.begin + kTile - 1) / kTile) % WAVES;
    attend_source(item.second, wave >= before ? wave - before : wave - before + WAVES);
  }

  // ---- join the waves.  More than four: the upper four hand their state to the four below them, lane by lane.
  if constexpr (WAVES > kJoined) {
    static_assert(RT == 1 && WAVES % kJoined == 0, "");
#pragma unroll
    for (int from = WAVES - kJoined; from >= kJoined; from -= kJoined) {
      const int slot = wave & (kJoined - 1);
      if (from + kJoined < WAVES) __syncthreads();
      if (wave >= from && wave < from + kJoined) {
#pragma unroll
        for (int c = 0; c < 8; ++c) *(f32x4*)&sh.acc[slot][n][32 * j + 4 * c] = rows.acc[0][c];
        sh.state[slot][lane][0] = rows.m_ref[0];
        sh.state[slot][lane][1] = rows.l_run[0];
        sh.state[slot][lane][2] = rows.cap;
      }
      __syncthreads();
      if (wave >= from - kJoined && wave < from) {
        const float m_other = sh.state[slot][lane][0], m = fmaxf(rows.m_ref[0], m_other);
        const float fa = __builtin_amdgcn_exp2f(rows.m_ref[0] - m), fb = __builtin_amdgcn_exp2f(m_other - m);
        rows.l_run[0] = rows.l_run[0] * fa + sh.state[slot][lane][1] * fb;
        rows.m_ref[0] = m;
        float ga = fa, gb = fb;
        if constexpr (kQuantised<FMT>) {
          const float cap_other = sh.state[slot][lane][2], both = fmaxf(rows.cap, cap_other);
          ga *= rows.cap / both;
          gb *= cap_other / both;
          rows.cap = both;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) rows.acc[0][c] = rows.acc[0][c] * ga + *(const f32x4*)&sh.acc[slot][n][32 * j + 4 * c] * gb;
      }
    }
    __syncthreads();
  }
  // Sixteen query rows at a time, normalised.
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float l = sum_over_quarters(rows.l_run[r]);
    const float norm = (l > 0.0f || l != l ? 1.0f / l : 0.0f) * (kQuantised<FMT> ? rows.cap : 1.0f);   // (an empty wave holds zeros)
    if (r) __syncthreads();
    if (wave < kJoined) {
      if (j == 0) {
        sh.m[wave][n] = rows.m_ref[r];
        sh.l[wave][n] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* to = &sh.acc[wave][n][32 * j + 8 * i];
        *(f32x4*)to = (f32x4){rows.acc[r][0][i], rows.acc[r][1][i], rows.acc[r][2][i], rows.acc[r][3][i]} * norm;
        *(f32x4*)(to + 4) = (f32x4){rows.acc[r][4][i], rows.acc[r][5][i], rows.acc[r][6][i], rows.acc[r][7][i]} * norm;
      }
    }
    __syncthreads();
    // sixteen threads a row, eight dims each (JOIN: all 256 share the `group` rows)
    const int slot = JOIN ? (tid >> 4) & (group - 1) : tid >> 4, d0 = 8 * (tid & 15);
    const int row = item.row0 + 16 * r + slot;
    if (tid < 16 * 16 && row < item.row_end) {
      float M = kNoReference, w[kJoined], L = 0.0f;   // w: l 2^(m - M) of the waves
#pragma unroll
      for (int x = 0; x < kJoined; ++x) M = fmaxf(M, sh.m[x][slot]);
      f32x4 lo = (f32x4){0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
      for (int x = 0; x < kJoined; ++x) {
        w[x] = sh.l[x][slot] * __builtin_amdgcn_exp2f(sh.m[x][slot] - M);   // (0 without rows)
        L += w[x];
      }
      const bool some = L > 0.0f || L != L;
      const float inv = some ? 1.0f / L : 0.0f;
#pragma unroll
      for (int x = 0; x < kJoined; ++x) {
        lo += *(const f32x4*)&sh.acc[x][slot][d0] * (w[x] * inv);
        hi += *(const f32x4*)&sh.acc[x][slot][d0 + 4] * (w[x] * inv);
      }
      if constexpr (JOIN) {
        static_assert(RT == 1 && WAVES == kJoined, "");
        join_shared(p, item.b0, item.h * group + slot, d0, tid >> 4, tid >> 4 >> p.group_log2, 16 >> p.group_log2, lo, hi,
                    M == kNoReference ? M : M - kWeightLog2<Rows<DT, FMT, RT>::kPF16>, L, sh.acc[0]);
        return;
      }
      store_result<Rows<DT, FMT, RT>::kPF16>(p, item.b0 + (row >> p.group_log2), item.h * group + (row & (group - 1)), item.slot, d0, lo, hi, M, L);
    }
  }
}

__device__ __forceinline__ void point_at(const KvRows& rows, int b, int h, AttendSource* src) {
  src->k = rows.k + b * rows.stride_b + h * rows.stride_h;
  src->v = rows.v + b * rows.stride_b + h * rows.stride_h;
  src->ks = rows.ks + b * rows.scale_b + h * rows.scale_h;
  src->vs = rows.vs + b * rows.scale_b + h * rows.scale_h;
  src->stride_n = rows.stride_n;
  src->scale_n = rows.scale_n;
  src->idx = nullptr;
}

__device__ __forceinline__ void take_shared(const KvAttendParams& p, int split, int h, AttendSource* src) {
  point_at(p.shared, 0, h, src);
  src->len = (int)p.shared.rows;
  src->begin = split * p.shared_tps;   // (below the rows)
  src->end = src->begin + min(src->len - src->begin, p.shared_tps);
}

template <bool INDEXED>
__device__ __forceinline__ void take_own(const KvAttendParams& p, int split, int b, int h, AttendSource* src) {
  point_at(p.own, b, h, src);
  src->len = (int)p.own.rows;
  if (p.own_len) src->len = __builtin_amdgcn_readfirstlane(max(min(p.own_len[b], src->len), 0));
  int count = src->len;
  if (INDEXED) {
    const int64_t seg = (int64_t)b * p.num_kv_heads + h;
    src->idx = p.kv_idx + seg * p.idx_len;
    count = p.kv_count ? __builtin_amdgcn_readfirstlane(max(min(p.kv_count[seg], p.idx_len), 0)) : p.idx_len;
  }
  src->begin = split * p.own_tps;      // (below the capacity; the length may end before it)
  src->end = src->begin + min(count - src->begin, p.own_tps);
}

// The own items of a launch: splits of (entry, head) pairs.
template <int DT, int FMT, bool INDEXED, int WAVES>
__device__ __forceinline__ void attend_own(const KvAttendParams& p, uint32_t own, AttendLds& sh, int32_t* sh_ids) {
  const uint32_t split = own % (uint32_t)p.own_splits, seg = own / (uint32_t)p.own_splits;
  AttendItem item;
  item.two = false;
  item.b0 = (int)(seg / (uint32_t)p.num_kv_heads);
  item.h = (int)(seg % (uint32_t)p.num_kv_heads);
  item.row0 = 0;
  item.row_end = 1 << p.group_log2;
  item.slot = p.shared_splits + (int)split;
  take_own<INDEXED>(p, (int)split, item.b0, item.h, &item.first);
  attend<DT, FMT, 1, INDEXED, WAVES>(p, item, sh, sh_ids);
}

// RT: sixteens of query rows that a workgroup of the shared source takes (0: there is no shared source).  Each wave holds all of them and
// has its tiles to itself: nothing is exchanged before the join.  RT = 4 takes the registers of a whole SIMD, RT = 2 those of a half.
template <int DT, int FMT, int RT, bool INDEXED>
__global__ __launch_bounds__(kThreads, RT >= 4 ? 1 : (RT == 2 ? 2 : 3)) void kv_attend_kernel(KvAttendParams p) {
  __shared__ AttendLds sh;
  __shared__ __align__(16) int32_t sh_ids[INDEXED ? kStagedIds : 4];
  const uint32_t shared_items = RT ? (uint32_t)(p.row_blocks * p.num_kv_heads * p.shared_splits) : 0u;
  AttendItem item;
  item.two = false;
  if (RT && blockIdx.x < shared_items) {
    const uint32_t split = blockIdx.x % (uint32_t)p.shared_splits, rest = blockIdx.x / (uint32_t)p.shared_splits;
    item.h = (int)(rest % (uint32_t)p.num_kv_heads);
    item.row0 = (int)(rest / (uint32_t)p.num_kv_heads) * 16 * RT;
    item.row_end = p.batch << p.group_log2;
    item.b0 = 0;
    item.slot = (int)split;
    take_shared(p, (int)split, item.h, &item.first);
    attend<DT, FMT, RT ? RT : 1, false, kWaves>(p, item, sh, sh_ids);
    return;
  }
  attend_own<DT, FMT, INDEXED, kWaves>(p, blockIdx.x - shared_items, sh, sh_ids);
}

// More query rows than a wave can hold: the waves of a workgroup take 32 query rows of a head each and go through the tokens together,
// a set of WAVES / 2 tiles at a time.  One half of the waves loads, converts and transposes the tiles of the even sets into matrix
// operands and leaves those in LDS, the other half those of the odd sets, each one set ahead, so that of the two waves of a SIMD one
// converts while the other multiplies and a set takes one barrier; all waves read all operands (8 KB of keys and 8 of values a tile).
// 64 x 8 x 8 query rows over 32768 + 256 rows of e4m3, bf16: 97 to 99 us in both launches, 705 TFLOP/s of products (with all waves
// converting eight tiles at a time, and two barriers, 106); int8 96; fp16, whose weights are in two parts: e4m3 116, int8 122.  What
// bounds it is the issue: its matrix units are busy 36 % of the 88 us and its vector units half of them; a wave issues, waits to
// issue, and waits for operands or a barrier a third of its time each.
template <int DT, int FMT, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void kv_attend_wide_kernel(KvAttendParams p) {
  static_assert(kQuantised<FMT>, "");
  using State = Rows<DT, FMT, 2>;
  constexpr int kSet = WAVES / 2;   // tiles of a set
  // Value operands with their scales in them, over a power of two of the tile, which saves a product for every weight.  e4m3: of
  // a scale only the power of two at or above it, so that the operands are exact (but for what lies 2^-24 below the tile's
  // largest); the rest of it, in (1/2, 1] (below 2 for scales beyond 2^127), goes to the weights in fp32 in the tiles where it is
  // not 1 throughout (it is 1 for what tka_kvq_write makes; 64 x 8 x 8 over 32768 rows with other scales: fp16 115 -> 121 us,
  // bf16 97 -> 99).  int8, whose scales are hardly ever powers of two, with bf16 queries: the whole scale, off by half a step of
  // fp16 twice (2^-10 of a value, below the 2^-8 of a bf16 output).  int8 with fp16 queries: the weights, which are then kept in
  // two parts, take the scales.
  constexpr bool kPowers = FMT == TKA_KV_E4M3, kScaled = kPowers || !State::kSplit;
  struct Operands {
    u32x4 frag[kSet][16][kWave];   // of a 32-token tile: K (x, kb) at 4 x + kb, V^T of dim c at 8 + c
    float ks[kSet][kTile], vs[kSet][kTile];
    float rest[kPowers ? kSet : 1][kTile];
    f32x2 tile_scale[kSet];        // and whether `rest` has anything but ones
  };
  __shared__ union {
    Operands sets[2];
    AttendLds join;
  } sh;
  const uint32_t shared_items = (uint32_t)(p.row_blocks * p.num_kv_heads * p.shared_splits);
  if (blockIdx.x >= shared_items) {
    attend_own<DT, FMT, false, WAVES>(p, blockIdx.x - shared_items, sh.join, nullptr);
    return;
  }
  const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t split = blockIdx.x % (uint32_t)p.shared_splits, rest_id = blockIdx.x / (uint32_t)p.shared_splits;
  const int h = (int)(rest_id % (uint32_t)p.num_kv_heads);
  const int row0 = (int)(rest_id / (uint32_t)p.num_kv_heads) * (32 * WAVES) + 32 * wave, row_end = p.batch << p.group_log2;
  AttendSource it;
  take_shared(p, (int)split, h, &it);
  State rows;
  rows.begin(p, 0, h, row0, row_end);
  const bool idle = row0 >= row_end;   // (it still loads its share)

  KTile<FMT> kt[2];
  VRow<FMT> vr[8];
  float scale = 0.0f;   // of a key row (lanes 0 .. 31) or a value row
  const auto load = [&](int tile) {
    if (tile < it.end) {
      const int start = tile_start(tile, it.end);
      DenseTiles<FMT> dense;
      AttendSource from = it;
      asm("" : "+s"(from.stride_n), "+s"(from.end));   // (the offsets are made here, not kept in registers over the loop)
      dense.begin(from);
      dense.key_rows(it, start, kt);
      dense.template value_rows<false>(it, start, vr);
      scale = (lane < kTile ? it.ks : it.vs)[(int64_t)(start + min(lane & (kTile - 1), dense.last)) * it.scale_n];
    }
  };
  const int half = wave / kSet, place = wave % kSet;   // this wave converts tile `place` of every other set
  // the operands of the tile in the registers, from position `tile` on
  const auto stage = [&](int tile, Operands& of) {
    const int token = lane & (kTile - 1);
    const bool cut = it.end - tile < kTile;
    const int start = tile_start(tile, it.end);
    hold<FMT>(kt, vr);
    if (cut) clear_masked<FMT>(tile_mask(start, tile, it.end), vr);
    u32x4 factor;   // of the value rows: pairs of slots
    if constexpr (kScaled) {
      float top = lane < kTile ? 0.0f : fabsf(scale);
#pragma unroll
      for (int x = 1; x < kTile; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, kWave));
      top = power_above(__shfl(top, kWave - 1, kWave));
      const float unit = power_inverse(top);
      const bool there = !cut || (start + token >= tile && start + token < it.end);
      _Float16 f = (_Float16)(scale * unit);
      bool uneven = false;
      if constexpr (kPowers) {
        const float power = power_at(scale);
        const float rest = there ? __builtin_ldexpf(fabsf(scale), 127 - (int)(__builtin_bit_cast(uint32_t, power) >> 23)) : 1.0f;
        f = (_Float16)(__builtin_copysignf(power, scale) * unit);
        uneven = __ballot(lane >= kTile && rest != 1.0f) != 0ull;
        if (lane >= kTile) of.rest[place][token] = rest;
      }
      if (!there) f = (_Float16)0.0f;
      _Float16* held = (_Float16*)of.vs[place];
      if (lane >= kTile) held[token] = f;
      if (lane == 0) of.tile_scale[place] = (f32x2){top, uneven ? 1.0f : 0.0f};
      wave_exchange();
      const u32x2 lo = *(const u32x2*)(held + 4 * j), hi = *(const u32x2*)(held + 16 + 4 * j);
      factor = (u32x4){lo[0], lo[1], hi[0], hi[1]};
      if (lane < kTile) of.ks[place][token] = scale * p.scale_log2e;
    } else {
      (lane < kTile ? of.ks : of.vs)[place][token] = lane < kTile ? scale * p.scale_log2e : scale;
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        of.frag[place][4 * x + kb][lane] = k_frag<FMT, State::kQF16>(kt[x], kb);
        __builtin_amdgcn_sched_barrier(0);   // (one operand after the other: all at once they do not fit the registers)
      }
    const auto values = [&](auto d) {
      constexpr int D = decltype(d)::value;
      u32x4 even, odd;
      v_frags<FMT, D>(vr, &even, &odd);
      if constexpr (kScaled) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          even[w] = as_bits(as_f16(even[w]) * as_f16(factor[w]));
          odd[w] = as_bits(as_f16(odd[w]) * as_f16(factor[w]));
        }
      }
      of.frag[place][8 + 2 * D][lane] = even;
      of.frag[place][9 + 2 * D][lane] = odd;
      __builtin_amdgcn_sched_barrier(0);
    };
    values(std::integral_constant<int, 0>());
    values(std::integral_constant<int, 1>());
    values(std::integral_constant<int, 2>());
    values(std::integral_constant<int, 3>());
  };

  const auto first_of = [&](int set) { return it.begin + (set * kSet + place) * kTile; };
  const int tiles = (it.end - it.begin + kTile - 1) / kTile, num_sets = (tiles + kSet - 1) / kSet;
  load(first_of(half));
  if (half == 0) {
    if (first_of(0) < it.end) stage(first_of(0), sh.sets[0]);
    load(first_of(2));
  }
  __syncthreads();
  for (int set = 0; set < num_sets; ++set, __syncthreads()) {
    if (((set + 1) & 1) == half && set + 1 < num_sets) {
      __builtin_amdgcn_s_setprio(1);   // (the others wait for it at the end of the set: 97.0 -> 96.2 us)
      if (first_of(set + 1) < it.end) stage(first_of(set + 1), sh.sets[(set + 1) & 1]);
      __builtin_amdgcn_s_setprio(0);
      load(first_of(set + 3));
    }
    if (idle) continue;
    const Operands& of = sh.sets[set & 1];
    const int count = min(tiles - set * kSet, kSet);
    u32x4 vfr[8];
    for (int t = 0; t < count; ++t) {
      const int tile = it.begin + (set * kSet + t) * kTile;
      const bool cut = it.end - tile < kTile;
      f32x4 sc[2][2];
      rows.scores(sc, [&](int x, int kb) { return of.frag[t][4 * x + kb][lane]; });
      float kf[8], vf[8], tile_scale = 0.0f;
      bool uneven = false;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const f32x4 a = *(const f32x4*)&of.ks[t][16 * x + 4 * j], b = kScaled ? a : *(const f32x4*)&of.vs[t][16 * x + 4 * j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kf[4 * x + i] = a[i];
          vf[4 * x + i] = b[i];
        }
      }
      if constexpr (kScaled) {
        const f32x2 held = of.tile_scale[t];
        const float top = held[0], flag = held[1];
        tile_scale = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, top)));
        if constexpr (kPowers) uneven = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, flag)) != 0;
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) vfr[x] = of.frag[t][8 + x][lane];   // (on their way during the softmax: 99 -> 97 us)
      __builtin_amdgcn_sched_barrier(0);
      rows.template attend<kScaled>(sc, kf, vf, tile_scale, uneven, of.rest[kPowers ? t : 0], cut ? tile_mask(tile_start(tile, it.end), tile, it.end) : 0u, cut,
                                    [&](auto d, u32x4* even, u32x4* odd) {
                                      constexpr int D = decltype(d)::value;
                                      *even = vfr[2 * D];
                                      *odd = vfr[2 * D + 1];
                                    });
    }
  }
  // each wave has its rows to itself: lane (n, j) dims 32 j .. 32 j + 31 of row n
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float l = sum_over_quarters(rows.l_run[r]);
    const float norm = (l > 0.0f || l != l ? 1.0f / l : 0.0f) * rows.cap;
    const int row = row0 + 16 * r + n;
    if (row < row_end) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store_result<State::kPF16>(p, row >> p.group_log2, (h << p.group_log2) + (row & ((1 << p.group_log2) - 1)), (int)split, 32 * j + 8 * i,
                                   (f32x4){rows.acc[r][0][i], rows.acc[r][1][i], rows.acc[r][2][i], rows.acc[r][3][i]} * norm,
                                   (f32x4){rows.acc[r][4][i], rows.acc[r][5][i], rows.acc[r][6][i], rows.acc[r][7][i]} * norm, rows.m_ref[r], l);
    }
  }
}

// Short calls: one workgroup of eight waves per (entry, head) attends to everything and writes the result, one launch.  The
// shared rows are then read for each entry.  Bound by the launch: one sequence, 8 heads, 256 rows 6.3 us (split and joined 7.8).
constexpr int kSoloWaves = 8;
template <int DT, int FMT, bool SHARED, bool INDEXED>
__global__ __launch_bounds__(kSoloWaves * kWave, 2) void kv_attend_solo_kernel(KvAttendParams p) {
  __shared__ AttendLds sh;
  __shared__ __align__(16) int32_t sh_ids[INDEXED ? kStagedIds : 4];
  AttendItem item;
  item.b0 = (int)(blockIdx.x / (uint32_t)p.num_kv_heads);
  item.h = (int)(blockIdx.x % (uint32_t)p.num_kv_heads);
  item.row0 = 0;
  item.row_end = 1 << p.group_log2;
  item.slot = 0;
  item.two = false;
  if constexpr (SHARED) {
    take_shared(p, 0, item.h, &item.first);
    item.two = p.own_splits != 0;
    if (item.two) take_own<false>(p, 0, item.b0, item.h, &item.second);
  } else {
    take_own<INDEXED>(p, 0, item.b0, item.h, &item.first);
  }
  attend<DT, FMT, 1, INDEXED, kSoloWaves>(p, item, sh, sh_ids);
}

// The second launch of calls with many short suffixes behind blocks of 256 query rows: a workgroup attends to the suffix of an (entry,
// head) and joins it with the partials of the prefix.
template <int DT, int FMT>
__global__ __launch_bounds__(kThreads, 3) void kv_attend_join_kernel(KvAttendParams p) {
  __shared__ AttendLds sh;
  AttendItem item;
  item.two = false;
  item.b0 = (int)(blockIdx.x / (uint32_t)p.num_kv_heads);
  item.h = (int)(blockIdx.x % (uint32_t)p.num_kv_heads);
  item.row0 = 0;
  item.row_end = 1 << p.group_log2;
  item.slot = 0;
  take_own<false>(p, 0, item.b0, item.h, &item.first);
  attend<DT, FMT, 1, false, kWaves, true>(p, item, sh, nullptr);
}

// The join of the splits, bound by the launch and by the partials (516 bytes each): 2.4 us for 8 rows of 8 splits, 4.2 us for 512 rows of
// 16 to 34.  One workgroup per query row: 32 lanes hold the 128 dims, eight groups of them take every eighth split.  A row whose sum is
// NaN stays NaN (an empty split holds zeros, so nothing has to be skipped); one without any key gets zeros and -infinity.
constexpr int kCombineGroups = kThreads / 32;
__global__ __launch_bounds__(kThreads) void kv_combine_kernel(KvAttendParams p) {
  __shared__ f32x4 sh_o[kCombineGroups][32];
  const int64_t row = blockIdx.x;
  const int g = threadIdx.x >> 5, d = threadIdx.x & 31, S = p.num_splits;
  const f32x2* ml = p.part_ml + row * S;
  const f32x4* pa = (const f32x4*)(p.part_acc + row * S * kHeadDim) + d;
  float M = kNoReference;
  for (int s = d; s < S; s += 32) M = fmaxf(M, ml[s][0]);   // (every group reads all references and sums: a line or two)
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
  float L = 0.0f;
  for (int s = d; s < S; s += 32) L += ml[s][1] * __builtin_amdgcn_exp2f(ml[s][0] - M);
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) L += __shfl_xor(L, x, 64);
  const bool some = L > 0.0f || L != L;
  const float inv = some ? 1.0f / L : 0.0f;
  f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int s0 = g; s0 < S; s0 += 4 * kCombineGroups) {
    f32x4 a[4];
    float w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * kCombineGroups, sc = s < S ? s : s0;
      a[u] = pa[(int64_t)sc * 32];
      w[u] = ml[sc][1] * __builtin_amdgcn_exp2f(ml[sc][0] - M) * inv;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + u * kCombineGroups < S) o += a[u] * w[u];
  }
  sh_o[g][d] = o;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  for (int x = 1; x < kCombineGroups; ++x) o += sh_o[x][d];
  const int hq = (int)(row % ((int64_t)p.num_kv_heads << p.group_log2));
  const int64_t b = row / ((int64_t)p.num_kv_heads << p.group_log2);
  u32x2 w;
  if (p.out_dtype == TKA_F16) w = (u32x2){pack_f16(o[0], o[1]), pack_f16(o[2], o[3])};
  else w = (u32x2){pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
  *(u32x2*)((uint16_t*)p.out + b * p.out_stride_b + (int64_t)hq * kHeadDim + 4 * d) = w;
  if (p.out_lse && d == 0) p.out_lse[row] = some ? (M + __builtin_log2f(L)) * 0.69314718055994531f : -INFINITY;
}

template <int DT, int FMT>
int launch_solo(const KvAttendParams& p, hipStream_t stream) {
  const uint32_t grid = (uint32_t)(p.batch * p.num_kv_heads);
  constexpr int threads = kSoloWaves * kWave;
  if (p.kv_idx) {
    if constexpr (kQuantised<FMT>) kv_attend_solo_kernel<DT, FMT, false, true><<<grid, threads, 0, stream>>>(p);
    else return TKA_EUNSUPPORTED;
  } else if (p.shared_splits) {
    kv_attend_solo_kernel<DT, FMT, true, false><<<grid, threads, 0, stream>>>(p);
  } else {
    kv_attend_solo_kernel<DT, FMT, false, false><<<grid, threads, 0, stream>>>(p);
  }
  return hip_status(hipGetLastError());
}

template <int DT, int FMT>
int launch_typed(const KvAttendParams& p, int row_tiles, hipStream_t stream) {
  if (row_tiles == 0) return launch_solo<DT, FMT>(p, stream);
  const uint32_t grid = (uint32_t)(p.row_blocks * p.num_kv_heads * p.shared_splits + p.batch * p.num_kv_heads * p.own_splits);
  if (p.kv_idx) {
    if constexpr (kQuantised<FMT>) kv_attend_kernel<DT, FMT, 0, true><<<grid, kThreads, 0, stream>>>(p);
    else return TKA_EUNSUPPORTED;
  } else if (!p.shared_splits) {
    kv_attend_kernel<DT, FMT, 0, false><<<grid, kThreads, 0, stream>>>(p);
  } else if (row_tiles == 1) {
    kv_attend_kernel<DT, FMT, 1, false><<<grid, kThreads, 0, stream>>>(p);
  } else if (row_tiles == 2) {
    kv_attend_kernel<DT, FMT, 2, false><<<grid, kThreads, 0, stream>>>(p);
  } else if (row_tiles == 4) {
    kv_attend_kernel<DT, FMT, 4, false><<<grid, kThreads, 0, stream>>>(p);
  } else {
    if constexpr (kQuantised<FMT>) {
      if (row_tiles == 8) kv_attend_wide_kernel<DT, FMT, 4><<<grid, 4 * kWave, 0, stream>>>(p);
      else kv_attend_wide_kernel<DT, FMT, 8><<<grid, 8 * kWave, 0, stream>>>(p);
    } else {
      return TKA_EUNSUPPORTED;
    }
  }
  return hip_status(hipGetLastError());
}

template <int DT>
int launch_format(const KvAttendParams& p, int format, int row_tiles, hipStream_t stream) {
  switch (format) {
    case TKA_KV_16BIT: return launch_typed<DT, TKA_KV_16BIT>(p, row_tiles, stream);
    case TKA_KV_E4M3: return launch_typed<DT, TKA_KV_E4M3>(p, row_tiles, stream);
    default: return launch_typed<DT, TKA_KV_INT8>(p, row_tiles, stream);
  }
}

}  // namespace

int launch_kv_attend(const KvAttendParams& p, int dtype, int format, int row_tiles, hipStream_t stream) {
  LaunchTimer timer(p.shared_splits ? "prefix_attend" : (p.kv_idx ? "kvq_attend_indexed" : "kvq_attend_dense"), stream);
  return dtype == TKA_F16 ? launch_format<TKA_F16>(p, format, row_tiles, stream) : launch_format<TKA_BF16>(p, format, row_tiles, stream);
}

namespace {
template <int DT>
int launch_join_format(const KvAttendParams& p, int format, hipStream_t stream) {
  const uint32_t grid = (uint32_t)(p.batch * p.num_kv_heads);
  switch (format) {
    case TKA_KV_E4M3: kv_attend_join_kernel<DT, TKA_KV_E4M3><<<grid, kThreads, 0, stream>>>(p); break;
    case TKA_KV_INT8: kv_attend_join_kernel<DT, TKA_KV_INT8><<<grid, kThreads, 0, stream>>>(p); break;
    default: return TKA_EUNSUPPORTED;
  }
  return hip_status(hipGetLastError());
}
}  // namespace

int launch_kv_attend_join(const KvAttendParams& p, int dtype, int format, hipStream_t stream) {
  LaunchTimer timer("prefix_suffix_join", stream);
  return dtype == TKA_F16 ? launch_join_format<TKA_F16>(p, format, stream) : launch_join_format<TKA_BF16>(p, format, stream);
}

int launch_kv_combine(const KvAttendParams& p, hipStream_t stream) {
  const uint32_t rows = (uint32_t)(p.batch * p.num_kv_heads) << p.group_log2;
  LaunchTimer timer("kv_combine", stream);
  kv_combine_kernel<<<rows, kThreads, 0, stream>>>(p);
  return hip_status(hipGetLastError());
}

}  // namespace tka
