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
// p * (scale / cap) * 2^14, with cap a power of two no scale seen so far exceeds (accumulators move with it), so that a
// weight is rounded by 2^-11 of itself down to 2^-28 of the largest, and by 2^-39 of that below.  16-bit rows: fp16
// weights are held the same way without a cap; bf16 weights have fp32's range but 8 bits only, the remainder goes through
// the matrix cores as a second operand, and they are held times 2^-32, so that no sum of the largest numbers overflows.
// (The factor sits in the exponent, and the sum of the weights has it too.)
//
// Results of waves and splits are joined normalised, out = sum (l_s 2^(m_s - M) / L) o_s: they stay in the range of V.
//
// A workgroup is one (source, batch entry or block of query rows, head, split); its waves take 32-token tiles in turn and
// are joined in LDS.  The shared source multiplies a block of 16 * RT query rows (entries x group) with each K / V tile.
#include <type_traits>

#include "kernels.hpp"
#include "kvq.hpp"

namespace tka {

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kTile = kAttendTile;
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
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const f16x2 v = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, v);
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
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);   // whole numbers below 2^8: the upper halves hold them
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

struct AttendLds {
  float acc[kWaves][16][kLdsRow];
  float m[kWaves][16];
  float l[kWaves][16];
};

template <bool F16>
constexpr float kWeightLog2 = F16 ? 14.0f : -32.0f;   // weights are held times 2^this

// What a workgroup attends to: positions [begin, end) of a source (of its token list where there is one) for the query
// rows [row0, row0 + 16 RT) below row_end; query row r is head h * group + r % group of batch entry b0 + r / group.
struct AttendItem {
  const unsigned char* k;   // of the entry and head
  const unsigned char* v;
  const float* ks;
  const float* vs;
  int64_t stride_n, scale_n;
  const int32_t* idx;
  int64_t len;              // rows of the cache that listed ids may name
  int64_t begin, end;
  int b0, h, row0, row_end, slot;
};

template <int DT, int FMT, int RT, bool INDEXED>
__device__ __forceinline__ void attend(const KvAttendParams& p, const AttendItem& it, AttendLds& sh) {
  constexpr bool kQF16 = DT == TKA_F16;
  constexpr bool kPF16 = kQuantised<FMT> || DT == TKA_F16;   // type of the second product
  constexpr bool kSplit = !kPF16 || DT == TKA_F16;           // weights in two parts
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int n = lane & 15, j = lane >> 4;
  const int group = 1 << p.group_log2;

  u32x4 qf[RT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = it.row0 + 16 * r + n;
    const bool there = row < it.row_end;
    const int rr = there ? row : 0;
    const uint16_t* q = (const uint16_t*)p.q + (int64_t)(it.b0 + (rr >> p.group_log2)) * p.q_stride_b +
                        (int64_t)(it.h * group + (rr & (group - 1))) * kHeadDim;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      qf[r][kb] = *(const u32x4*)(q + k_dim<FMT>(kb, j));
      if (!there) qf[r][kb] = (u32x4){0u, 0u, 0u, 0u};
    }
  }

  float m_run[RT], l_run[RT];   // of query row n of each tile; l_run: this quarter's share
  f32x4 acc[RT][8];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m_run[r] = -INFINITY;
    l_run[r] = 0.0f;
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[r][c] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  float cap = __builtin_bit_cast(float, 17u << 23);   // 2^-110: the least cap (its reciprocal stays in range)

  const unsigned char* kb_base = it.k + 16 * j;
  const unsigned char* vb_base = it.v + (kQuantised<FMT> ? 8 : 16) * n;

  for (int64_t tile = it.begin + wave * kTile; tile < it.end; tile += kWaves * kTile) {
    const bool full = tile + kTile <= it.end;
    int64_t tk[2], tv[8];
    bool ok[8];
    bool skipped = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int64_t pos = tile + 16 * x + n;
      const int64_t pc = pos < it.end ? pos : it.end - 1;
      int64_t t = INDEXED ? (int64_t)it.idx[pc] : pc;
      if (INDEXED && (t < 0 || t >= it.len)) t = 0;
      tk[x] = t;
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int64_t pos = tile + slot_token(j, s);
      ok[s] = pos < it.end;
      const int64_t pc = ok[s] ? pos : it.end - 1;
      int64_t t = INDEXED ? (int64_t)it.idx[pc] : pc;
      if (INDEXED && (t < 0 || t >= it.len)) {
        ok[s] = false;
        t = 0;
        skipped = true;
      }
      tv[s] = t;
    }
    KTile<FMT> kt[2];
    VRow<FMT> vr[8];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < KTile<FMT>::kLoads; ++y) kt[x].w[y] = *(const u32x4*)(kb_base + tk[x] * it.stride_n + 64 * y);
#pragma unroll
    for (int s = 0; s < 8; ++s) vr[s] = *(const VRow<FMT>*)(vb_base + tv[s] * it.stride_n);
    float ks[8], vs[8];
    if constexpr (kQuantised<FMT>) {
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        ks[s] = it.ks[tv[s] * it.scale_n];
        vs[s] = it.vs[tv[s] * it.scale_n];
      }
    }
    // rows of masked slots (behind the end, ids outside the cache) must not reach the products: 0 * inf, 0 * NaN
    if (!full || (INDEXED && __ballot(skipped) != 0ull)) {
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (!ok[s]) {
          vr[s] = VRow<FMT>{};
          if constexpr (kQuantised<FMT>) vs[s] = 0.0f;
        }
    }
    float weight[8];   // scale of a slot's value row over the cap
    if constexpr (kQuantised<FMT>) {
      float top = vs[0];
#pragma unroll
      for (int s = 1; s < 8; ++s) top = fmaxf(top, vs[s]);
      if (__ballot(top > cap) != 0ull) {
        top = max_over_quarters(top);
        const uint32_t e = (__builtin_bit_cast(uint32_t, top) + 0x7fffffu) & 0x7f800000u;   // the power of two at or above it
        const float raised = __builtin_bit_cast(float, e < 0x7f000000u ? e : 0x7f000000u);
        const float drop = cap / raised;
        cap = raised;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[r][c] *= drop;
      }
      const float unit = 1.0f / cap;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        weight[s] = vs[s] * unit;
        ks[s] *= p.scale_log2e;
      }
    }

    u32x4 pf[RT], pf_lo[RT];
    {
      f32x4 sc[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r) sc[r][0] = sc[r][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const u32x4 a = k_frag<FMT, kQF16>(kt[x], kb);
#pragma unroll
          for (int r = 0; r < RT; ++r) sc[r][x] = mfma<kQF16>(a, qf[r][kb], sc[r][x]);
        }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float xs[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          xs[s] = sc[r][s >> 2][s & 3] * (kQuantised<FMT> ? ks[s] : p.scale_log2e);
          if (!ok[s]) xs[s] = -INFINITY;
        }
        float top = xs[0];
#pragma unroll
        for (int s = 1; s < 8; ++s) top = fmaxf(top, xs[s]);
        top = max_over_quarters(top);
        const float m_new = fmaxf(m_run[r], top);
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;   // nothing but masked rows so far
        const float alpha = __builtin_amdgcn_exp2f(m_run[r] - m_use);
        float ps[8], sum = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          ps[s] = __builtin_amdgcn_exp2f(xs[s] - (m_use - kWeightLog2<kPF16>));
          sum += ps[s];
        }
        m_run[r] = m_new;
        l_run[r] = l_run[r] * alpha + sum;
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[r][c] *= alpha;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float a = ps[2 * w], b = ps[2 * w + 1];
          if constexpr (kPF16) {
            const float x = kQuantised<FMT> ? a * weight[2 * w] : a, y = kQuantised<FMT> ? b * weight[2 * w + 1] : b;
            pf[r][w] = pack_f16(x, y);
            if constexpr (kSplit) {
              uint32_t hi = pf[r][w];
              asm("" : "+v"(hi));   // (the compiler otherwise folds the conversions into mixed-precision multiply-adds and takes the first pair's rounded weights for all four)
              const f16x2 h = __builtin_bit_cast(f16x2, hi);
              pf_lo[r][w] = pack_f16(x - (float)h[0], y - (float)h[1]);
            }
          } else {
            pf[r][w] = pack_bf16(a, b);
            pf_lo[r][w] = pack_bf16(a - __builtin_bit_cast(float, pf[r][w] << 16), b - __builtin_bit_cast(float, pf[r][w] & 0xffff0000u));
          }
        }
      }
    }

    const auto values = [&](auto d) {
      constexpr int D = decltype(d)::value;
      u32x4 even, odd;
      v_frags<FMT, D>(vr, &even, &odd);
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

  // ---- join the waves, sixteen query rows at a time
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float l = sum_over_quarters(l_run[r]);
    const float norm = (l > 0.0f || l != l ? 1.0f / l : 0.0f) * (kQuantised<FMT> ? cap : 1.0f);   // (an empty wave holds zeros)
    if (r) __syncthreads();
    if (j == 0) {
      sh.m[wave][n] = m_run[r];
      sh.l[wave][n] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* to = &sh.acc[wave][n][32 * j + 8 * i];
      *(f32x4*)to = (f32x4){acc[r][0][i], acc[r][1][i], acc[r][2][i], acc[r][3][i]} * norm;
      *(f32x4*)(to + 4) = (f32x4){acc[r][4][i], acc[r][5][i], acc[r][6][i], acc[r][7][i]} * norm;
    }
    __syncthreads();
    // sixteen threads a row, eight dims each
    const int row = it.row0 + 16 * r + (tid >> 4), d0 = 8 * (tid & 15);
    if (row < it.row_end) {
      float M = -INFINITY, w[kWaves], L = 0.0f;   // w: l 2^(m - M) of the waves
#pragma unroll
      for (int x = 0; x < kWaves; ++x) M = fmaxf(M, sh.m[x][tid >> 4]);
      const float m_use = M == -INFINITY ? 0.0f : M;
      f32x4 lo = (f32x4){0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) {
        w[x] = sh.l[x][tid >> 4] * __builtin_amdgcn_exp2f(sh.m[x][tid >> 4] - m_use);
        L += w[x];
      }
      const bool some = L > 0.0f || L != L;
      const float inv = some ? 1.0f / L : 0.0f;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) {
        lo += *(const f32x4*)&sh.acc[x][tid >> 4][d0] * (w[x] * inv);
        hi += *(const f32x4*)&sh.acc[x][tid >> 4][d0 + 4] * (w[x] * inv);
      }
      const int b = it.b0 + (row >> p.group_log2), hq = it.h * group + (row & (group - 1));
      const int64_t flat = (int64_t)b * p.num_kv_heads * group + hq;
      if (p.num_splits > 1) {
        const int64_t slot = flat * p.num_splits + it.slot;
        f32x4* to = (f32x4*)(p.part_acc + slot * kHeadDim + d0);
        to[0] = lo;
        to[1] = hi;
        if (d0 == 0) {
          p.part_m[slot] = M - kWeightLog2<kPF16>;   // (the sum as it is held belongs to a maximum that much lower)
          p.part_l[slot] = L;
        }
      } else {
        u32x4 o;
        if (p.out_dtype == TKA_F16) o = (u32x4){pack_f16(lo[0], lo[1]), pack_f16(lo[2], lo[3]), pack_f16(hi[0], hi[1]), pack_f16(hi[2], hi[3])};
        else o = (u32x4){pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]), pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3])};
        *(u32x4*)((uint16_t*)p.out + b * p.out_stride_b + (int64_t)hq * kHeadDim + d0) = o;
        if (p.out_lse && d0 == 0) p.out_lse[flat] = some ? (M + (__builtin_log2f(L) - kWeightLog2<kPF16>)) * 0.69314718055994531f : -INFINITY;
      }
    }
  }
}

__device__ __forceinline__ void point_at(const KvRows& rows, int b, int h, AttendItem* it) {
  it->k = rows.k + b * rows.stride_b + h * rows.stride_h;
  it->v = rows.v + b * rows.stride_b + h * rows.stride_h;
  it->ks = rows.ks + b * rows.scale_b + h * rows.scale_h;
  it->vs = rows.vs + b * rows.scale_b + h * rows.scale_h;
  it->stride_n = rows.stride_n;
  it->scale_n = rows.scale_n;
}

// RT: sixteens of query rows that a workgroup of the shared source takes (0: there is no shared source)
template <int DT, int FMT, int RT, bool INDEXED>
__global__ __launch_bounds__(kThreads) void kv_attend_kernel(KvAttendParams p) {
  __shared__ AttendLds sh;
  const uint32_t shared_items = RT ? (uint32_t)(p.row_blocks * p.num_kv_heads * p.shared_splits) : 0u;
  AttendItem it;
  if (RT && blockIdx.x < shared_items) {
    const uint32_t split = blockIdx.x % (uint32_t)p.shared_splits, rest = blockIdx.x / (uint32_t)p.shared_splits;
    it.h = (int)(rest % (uint32_t)p.num_kv_heads);
    it.row0 = (int)(rest / (uint32_t)p.num_kv_heads) * 16 * RT;
    it.row_end = p.batch << p.group_log2;
    it.b0 = 0;
    it.idx = nullptr;
    it.len = p.shared.rows;
    it.begin = (int64_t)split * p.shared_tps;
    it.end = it.begin + p.shared_tps;
    it.end = it.end < it.len ? it.end : it.len;
    it.slot = (int)split;
    point_at(p.shared, 0, it.h, &it);
    attend<DT, FMT, RT ? RT : 1, false>(p, it, sh);
    return;
  }
  const uint32_t item = blockIdx.x - shared_items;
  const uint32_t split = item % (uint32_t)p.own_splits, seg = item / (uint32_t)p.own_splits;
  it.b0 = (int)(seg / (uint32_t)p.num_kv_heads);
  it.h = (int)(seg % (uint32_t)p.num_kv_heads);
  it.row0 = 0;
  it.row_end = 1 << p.group_log2;
  it.len = p.own.rows;
  if (p.own_len) {
    const int64_t len = p.own_len[it.b0];
    it.len = len < 0 ? 0 : (len < it.len ? len : it.len);
  }
  int64_t count = it.len;
  it.idx = nullptr;
  if (INDEXED) {
    it.idx = p.kv_idx + (int64_t)seg * p.idx_len;
    count = p.kv_count ? p.kv_count[seg] : p.idx_len;
    count = count < 0 ? 0 : (count < p.idx_len ? count : p.idx_len);
  }
  it.begin = (int64_t)split * p.own_tps;
  it.end = it.begin + p.own_tps;
  it.end = it.end < count ? it.end : count;
  it.slot = p.shared_splits + (int)split;
  point_at(p.own, it.b0, it.h, &it);
  attend<DT, FMT, 1, INDEXED>(p, it, sh);
}

// One workgroup per query row: 32 lanes hold the 128 dims, eight groups of them take every eighth split.  A row whose sum is
// NaN stays NaN (an empty split holds zeros, so nothing has to be skipped); one without any key gets zeros and -infinity.
constexpr int kCombineGroups = kThreads / 32;
__global__ __launch_bounds__(kThreads) void kv_combine_kernel(KvAttendParams p) {
  __shared__ f32x4 sh_o[kCombineGroups][32];
  const int64_t row = blockIdx.x;
  const int g = threadIdx.x >> 5, d = threadIdx.x & 31, S = p.num_splits;
  const float* pm = p.part_m + row * S;
  const float* pl = p.part_l + row * S;
  const f32x4* pa = (const f32x4*)(p.part_acc + row * S * kHeadDim) + d;
  float M = -INFINITY;
  for (int s = d; s < S; s += 32) M = fmaxf(M, pm[s]);   // (every group reads all maxima and sums: a line or two)
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
  const float m_use = M == -INFINITY ? 0.0f : M;
  float L = 0.0f;
  for (int s = d; s < S; s += 32) L += pl[s] * __builtin_amdgcn_exp2f(pm[s] - m_use);
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
      w[u] = pl[sc] * __builtin_amdgcn_exp2f(pm[sc] - m_use) * inv;
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
int launch_typed(const KvAttendParams& p, int row_tiles, uint32_t grid, hipStream_t stream) {
  if (p.kv_idx) {
    if constexpr (kQuantised<FMT>) kv_attend_kernel<DT, FMT, 0, true><<<grid, kThreads, 0, stream>>>(p);
    else return TKA_EUNSUPPORTED;
  } else if (!p.shared_splits) {
    kv_attend_kernel<DT, FMT, 0, false><<<grid, kThreads, 0, stream>>>(p);
  } else if (row_tiles == 1) {
    kv_attend_kernel<DT, FMT, 1, false><<<grid, kThreads, 0, stream>>>(p);
  } else if (row_tiles == 2) {
    kv_attend_kernel<DT, FMT, 2, false><<<grid, kThreads, 0, stream>>>(p);
  } else {
    kv_attend_kernel<DT, FMT, 4, false><<<grid, kThreads, 0, stream>>>(p);
  }
  return hip_status(hipGetLastError());
}

template <int DT>
int launch_format(const KvAttendParams& p, int format, int row_tiles, uint32_t grid, hipStream_t stream) {
  switch (format) {
    case TKA_KV_16BIT: return launch_typed<DT, TKA_KV_16BIT>(p, row_tiles, grid, stream);
    case TKA_KV_E4M3: return launch_typed<DT, TKA_KV_E4M3>(p, row_tiles, grid, stream);
    default: return launch_typed<DT, TKA_KV_INT8>(p, row_tiles, grid, stream);
  }
}

}  // namespace

int launch_kv_attend(const KvAttendParams& p, int dtype, int format, int row_tiles, hipStream_t stream) {
  const uint32_t grid = (uint32_t)(p.row_blocks * p.num_kv_heads * p.shared_splits + p.batch * p.num_kv_heads * p.own_splits);
  LaunchTimer timer(p.shared_splits ? "prefix_attend" : (p.kv_idx ? "kvq_attend_indexed" : "kvq_attend_dense"), stream);
  return dtype == TKA_F16 ? launch_format<TKA_F16>(p, format, row_tiles, grid, stream)
                          : launch_format<TKA_BF16>(p, format, row_tiles, grid, stream);
}

int launch_kv_combine(const KvAttendParams& p, hipStream_t stream) {
  const uint32_t rows = (uint32_t)(p.batch * p.num_kv_heads) << p.group_log2;
  LaunchTimer timer("kv_combine", stream);
  kv_combine_kernel<<<rows, kThreads, 0, stream>>>(p);
  return hip_status(hipGetLastError());
}

}  // namespace tka
