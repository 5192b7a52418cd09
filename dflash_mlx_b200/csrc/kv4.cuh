// Shared between the 4-bit KV cache kernels (kv4.cu: write, read, attention for few rows; kv4_tc.cu: for many).
#pragma once

#include "common.cuh"

namespace dflash {
namespace kv4 {

constexpr int kGroup = 64;   // channels per scale / bias

struct SdpaArgs {
  const void* q;
  long long q_sb, q_sh, q_st;
  dflash_kv4_cache k, v;
  const void* mask;
  int mask_kind;
  long long m_sb, m_sh, m_st, m_sn;
  void* out;
  float* part_o;   // [B*Hk*rows][splits][D], over the range's own sum (a sum of values may be no fp32 number), then part_m / part_l
  float* part_m;
  float* part_l;
  const int* lengths;
  int B, Hq, Hk, gqa, T, rows;   // rows = gqa * T query rows per (sequence, KV head); row r is position r / gqa, head r % gqa
  int max_length, splits;
  float scale;
};

// 2^x to 2^-22; results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / x to 2^-23, for sums of probabilities (at least about 1, or 0, NaN, +inf); 1 for the sum of nothing.
__device__ __forceinline__ float over_sum(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return x == 0.f ? 1.f : y;
}

// Offset of query / output row `r` of (b, hk) in the contiguous output [B,Hq,T,D], in rows.
__device__ __forceinline__ size_t out_row(const SdpaArgs& a, int b, int hk, int r) {
  const int t = r / a.gqa, h = hk * a.gqa + r % a.gqa;
  return ((size_t)b * a.Hq + h) * a.T + t;
}

// Mask value of (row, key) added to the scaled score t; -inf hides.
template <typename T>
__device__ __forceinline__ float apply_mask(const SdpaArgs& a, float t, long long at) {
  if (a.mask_kind == 1) return ((const uint8_t*)a.mask)[at] ? t : -INFINITY;
  const float m = a.mask_kind == 2 ? MmaTraits<T>::to_float(((const T*)a.mask)[at]) : ((const float*)a.mask)[at];
  return m == -INFINITY ? -INFINITY : t + m;   // a hidden key stays hidden whatever its score (NaN, +inf)
}

// kv4_tc.cu: the attention's pass over the keys for many rows per KV head (always above kFewRows; kTcRows rows a block), into the output or,
// with several splits, the partials.
constexpr int kFewRows = 16, kTcRows = 128;
int launch_partials_tc(const SdpaArgs& a, int dtype, int D, cudaStream_t st, int device);

}  // namespace kv4
}  // namespace dflash
