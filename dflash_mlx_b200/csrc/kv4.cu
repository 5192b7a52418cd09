// The 4-bit KV cache: quantising new rows as they are written, reading rows back, and softmax attention over the codes.
//
// Layout (that of mlx-lm's quantised cache and of this library's packed weights): per position D/8 words of eight codes, one
// scale and one bias per 64 channels; a channel stands for code * scale + bias.
//
// Attention over the codes, per KV head with rows = (Hq/Hk) * T query rows r and keys n, group g = 64 channels:
//   S[r,n] = scale * sum_g ( sk[n,g] * sum_{d in g} q[r,d] ck[n,d]  +  bk[n,g] * sum_{d in g} q[r,d] )
//   O[r,d] = sum_n p[r,n] sv[n,g] (cv[n,d] - 8)  +  sum_n p[r,n] (bv[n,g] + 8 sv[n,g])          (g the group of d)
// In the kernel of few rows below, the codes enter both products as exact small integers; scales and biases are applied in fp32
// around them, so the only rounding besides fp32 sums is that of p * sv to fp16 (11 bits; q is exact in fp16 but for elements far below
// its row's largest).  The kernel of many rows (kv4_tc.cu) rounds the cache's values to fp16 as well.
#include <mutex>

#include "kv4.cuh"

namespace dflash {
namespace kv4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---- write -------------------------------------------------------------------------------------------------------------
// A lane owns the eight channels of one word, eight lanes a group: minimum and maximum in three shuffles, no shared memory.
// Bound by instruction issue (prompts: 76 % of the slots while blocks run, HBM at a quarter of its rate) or by the launch (single
// tokens): a warp has its next row on the way under the current one, in a rolled loop (eight rows unrolled missed the instruction
// cache: 21 us for 2 x 4133 rows of 4 heads x 256, 17.9 now; its HBM floor is 7).  One token: 1.6 us.  blockIdx.x is (sequence,
// head), so no lane divides.
struct WriteArgs {
  const void* x[2];
  long long sb[2], sh[2], st[2];
  dflash_kv4_cache c[2];
  const int* offsets;
  const int* counts;
  int Hk, T, capacity, steps;   // steps: rows of a warp (times 256 / D)
};

// The code as a float, round((v - bias) / scale) in 0..15.  The quotient is that of an IEEE division: by the correctly rounded
// reciprocal and one correction by the exact residual (Markstein), as long as nothing in it is subnormal (`plain`).  bias is the
// group's minimum, so there is nothing below 0; a scale that was rounded down far (a subnormal) goes above 15.  Adding and
// taking away 1.5 * 2^23 rounds to a whole number, ties to even, without the slow conversion instructions.
__device__ __forceinline__ float code_of(float v, float bias, float scale, float inv, bool plain) {
  constexpr float kMagic = 12582912.f;
  const float y = __fsub_rn(v, bias);
  float q = y * inv;
  if (plain) q = __fmaf_rn(__fmaf_rn(-q, scale, y), inv, q);
  else q = __fdiv_rn(y, scale);
  return fminf(__fsub_rn(__fadd_rn(q, kMagic), kMagic), 15.f);
}
// x / 15 to the last bit for every value of the two 16-bit types (tested over all of them): the quotient by the rounded reciprocal
// and one correction by its residual.
__device__ __forceinline__ float by_15(float x) {
  constexpr float kInv = 1.f / 15.f;
  const float q = __fmul_rn(x, kInv);
  return __fmaf_rn(__fmaf_rn(-15.f, q, x), kInv, q);
}
__device__ __forceinline__ __nv_bfloat162 pair_of(uint32_t u, __nv_bfloat16) { return *(const __nv_bfloat162*)&u; }
__device__ __forceinline__ __half2 pair_of(uint32_t u, __half) { return *(const __half2*)&u; }

template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_write_kernel(const WriteArgs a, int* __restrict__ err) {
  using TR = MmaTraits<T>;
  constexpr int kLanes = D / 8, kPer = 32 / kLanes;   // lanes of a row, rows of a warp at once
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = blockIdx.z;
  const int j = lane % kLanes;
  const int b = blockIdx.x / a.Hk, h = blockIdx.x % a.Hk;
  const int n = min(a.counts ? a.counts[b] : a.T, a.T);
  const long long at = a.offsets[b];
  const T* x = (const T*)a.x[side] + b * a.sb[side] + h * a.sh[side] + 8 * j;
  const dflash_kv4_cache c = a.c[side];
  uint32_t* codes = c.codes + b * c.codes_batch_stride + h * c.codes_head_stride + j;
  T* scales = (T*)c.scales + b * c.scales_batch_stride + h * c.scales_head_stride + (j >> 3);
  T* biases = (T*)c.biases + b * c.biases_batch_stride + h * c.biases_head_stride + (j >> 3);
  const int first = (int)blockIdx.y * 4 * kPer * a.steps + warp * kPer + lane / kLanes;
  auto inside = [&](int t) { return t < n && at + t >= 0 && at + t < a.capacity; };
  auto load = [&](int t) { return inside(t) ? *(const uint4*)(x + t * a.st[side]) : make_uint4(0, 0, 0, 0); };
  uint4 next = load(first);
#pragma unroll 1
  for (int s = 0; s < a.steps; ++s) {
    const int t = first + s * 4 * kPer;
    const uint4 raw = next;
    if (s + 1 < a.steps) next = load(t + 4 * kPer);
    if (__all_sync(0xffffffffu, t >= n)) break;
    if (t < n && !inside(t) && j == 0) atomicCAS(err, 0, 61 | ((t & 0x7FFFFF) << 8));
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    // maximum and minimum in pairs; a NaN wins both
    const auto hi2 = __hmax2_nan(__hmax2_nan(pair_of(u[0], T()), pair_of(u[1], T())), __hmax2_nan(pair_of(u[2], T()), pair_of(u[3], T())));
    const auto lo2 = __hmin2_nan(__hmin2_nan(pair_of(u[0], T()), pair_of(u[1], T())), __hmin2_nan(pair_of(u[2], T()), pair_of(u[3], T())));
    const T hi_t = __hmax_nan(hi2.x, hi2.y), nlo_t = __hneg(__hmin_nan(lo2.x, lo2.y));
    uint32_t ext = (uint32_t) * (const uint16_t*)&hi_t | ((uint32_t) * (const uint16_t*)&nlo_t << 16);   // maximum, -minimum
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const auto m = __hmax2_nan(pair_of(ext, T()), pair_of(__shfl_xor_sync(0xffffffffu, ext, o), T()));
      ext = *(const uint32_t*)&m;
    }
    const float hi = TR::bits_to_float((uint16_t)ext), lo = -TR::bits_to_float((uint16_t)(ext >> 16));
    // NaN as soon as one value is NaN or infinite
    const float bad = fmaf(hi, 0.f, lo * 0.f);
    // subnormals count too: the codes are defined to the last bit (this file is compiled without fast math)
    const T scale_t = TR::from_float(__fadd_rn(__fsub_rn(by_15(hi), by_15(lo)), bad));
    const T bias_t = TR::from_float(__fadd_rn(lo, bad));
    const float scale = TR::to_float(scale_t), bias = TR::to_float(bias_t);
    uint32_t word = 0;
    if (scale > 0.f) {
      const float inv = __frcp_rn(scale);
      float f[2];   // four codes each, as one whole number below 2^16
      auto codes_of = [&](bool plain) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float k[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            k[e] = code_of(TR::bits_to_float((uint16_t)(u[2 * w + (e >> 1)] >> (16 * (e & 1)))), bias, scale, inv, plain);
          f[w] = fmaf(fmaf(fmaf(k[3], 16.f, k[2]), 16.f, k[1]), 16.f, k[0]) + 8388608.f;
        }
      };
      if (scale > 0x1p-80f && scale < 0x1p100f) codes_of(true);
      else codes_of(false);
      word = prmt(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x5410);
    }
    if (inside(t)) {
      const long long p = at + t;
      codes[p * (D / 8)] = word;
      if ((j & 7) == 0) {
        scales[p * (D / kGroup)] = scale_t;
        biases[p * (D / kGroup)] = bias_t;
      }
    }
  }
}

// ---- read --------------------------------------------------------------------------------------------------------------
struct ReadArgs {
  dflash_kv4_cache c[2];
  void* out[2];
  const int* starts;
  int start, Hk, T, capacity;
};

// The same split as the write: a lane unpacks one word into 16 bytes of output.  65537 rows of 4 heads x 256: 57 us, 6.0 TB/s.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(128) kv4_read_kernel(const ReadArgs a) {
  using TR = MmaTraits<T>;
  constexpr int kLanes = D / 8, kPer = 32 / kLanes, kBlock = 4 * kPer * kRows;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = blockIdx.z;
  const int j = lane % kLanes;
  const int b = blockIdx.x / a.Hk, h = blockIdx.x % a.Hk;
  const long long at = a.starts ? a.starts[b] : a.start;
  const dflash_kv4_cache c = a.c[side];
  const uint32_t* codes = c.codes + b * c.codes_batch_stride + h * c.codes_head_stride + j;
  const T* scales = (const T*)c.scales + b * c.scales_batch_stride + h * c.scales_head_stride + (j >> 3);
  const T* biases = (const T*)c.biases + b * c.biases_batch_stride + h * c.biases_head_stride + (j >> 3);
  T* out = (T*)a.out[side] + (long long)blockIdx.x * a.T * D + 8 * j;
  for (int t0 = blockIdx.y * kBlock; t0 < a.T; t0 += gridDim.y * kBlock) {
    uint32_t word[kRows];
    T scale[kRows], bias[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int t = t0 + (warp * kRows + i) * kPer + lane / kLanes;
      const long long p = at + t;
      word[i] = 0;
      scale[i] = bias[i] = TR::from_float(0.f);
      if (t < a.T && p >= 0 && p < a.capacity) {
        word[i] = codes[p * (D / 8)];
        scale[i] = scales[p * (D / kGroup)];
        bias[i] = biases[p * (D / kGroup)];
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int t = t0 + (warp * kRows + i) * kPer + lane / kLanes;
      if (t < a.T) {
        const float s = TR::to_float(scale[i]), z = TR::to_float(bias[i]);
        uint4 o;
        uint32_t* po = (uint32_t*)&o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // code * scale is exact in fp32 (4 + 11 bits), so there is one rounding in the sum and one to the output type
          const T x0 = TR::from_float(fmaf((float)((word[i] >> (8 * e)) & 15u), s, z));
          const T x1 = TR::from_float(fmaf((float)((word[i] >> (8 * e + 4)) & 15u), s, z));
          po[e] = (uint32_t) * (const uint16_t*)&x0 | ((uint32_t) * (const uint16_t*)&x1 << 16);
        }
        *(uint4*)(out + (long long)t * D) = o;
      }
    }
  }
}

// ---- attention, few rows per KV head -----------------------------------------------------------------------------------
// One warp works on 16 keys at a time, on its own: codes and scales of its next tiles arrive by cp.async in a ring of
// kStages shared-memory buffers that only this warp touches, so there is no block-wide barrier in the loop.  Both products
// have the KEYS' codes (or their transpose) as the 16-row operand and 8 query rows as the 8 columns, so one decoded token of a
// grouped model (Hq/Hk <= 8 rows) wastes nothing:
//   S^T [16 keys, 8 rows] += K codes [16, 16 channels] x Q^T : a thread unpacks the two words of its quarter of a group; the
//       16 channels of an MMA step are any 16 of one group (Q is laid out to match), so a group's sum ends in its own
//       accumulator and takes its scale there.
//   O^T [16 channels, 8 rows] += V codes^T [16, 16 keys] x P' : P' = p * sv in fp16 (11 bits; fp32's would need four times the
//       MMAs).  Nibble t and 4 + t of a word are rows r and r + 8 of MMA t, so a thread's words serve four MMAs without crossing
//       lanes.
// P' in fp16's range, whatever the scales, and without a row noticing keys that it does not see: a key whose largest |sv| lies in
// [2^-7, 2^3) is multiplied by 2^8 like all of its kind, so P' <= 2^15, and probabilities down to 2^-17 of the largest keep 9 bits under
// the smallest of these scales; any other key by a power of two of its own, 2^(8 - x), which P' and the row's exponent take back:
// P' = p sv 2^(8 - ev), ev = 0 until the row sees such a key.  A tile without one, under rows with ev = 0, does not touch any of this.
// Codes become exact fp16 integers by OR-ing the nibble into 1024 and one packed operation that takes the constant away again
// (left in, a sum would carry 1024 times sum |q| or sum P', which costs digits); values are centred as code - 8, which halves
// what the rounding of P' is multiplied with.  q is brought to fp16 by a power of two per row: bf16's 8 bits are exact in it
// down to 2^-28 of the row's largest element.
// The running maximum moves only when a score exceeds it by 4 octaves (p <= 16 otherwise), so the accumulators are rarely
// rescaled.  The warps of a block and then the splits of the key range are merged with fp32 partials.
// Measured (D = 256, bf16): 8 rows, 16 ragged sequences up to 32768: 71.5 us, 2.9 TB/s, with 58 % of the issue slots and half of the ALU pipe
// busy while blocks run and a sixth of the time behind the longest sequence; 6 rows over 4097 positions: 9.1 us with the combine.
// Warps of a block.  Two blocks share an SM, so that one starts or merges while the other streams; as many warps as the registers
// allow (the loop is bound by instruction issue: unpacking, scales and softmax next to the MMAs).
constexpr int kStages = 3;   // tiles of a warp in shared memory
template <int D, int NT> constexpr int kWarpsOf = NT == 2 ? (D == 256 ? 4 : 6) : (D == 256 ? 6 : 8);
constexpr float kLn2 = 0.6931471805599453f, kMaxStep = 4 * kLn2;
constexpr float kUsual = 256.f;            // the power of two of usual value scales
__device__ __forceinline__ bool unusual(float big) {   // outside [2^-7, 2^3), and not 0
  const uint32_t u = __float_as_uint(big);
  return u - (120u << 23) >= (10u << 23) && u != 0;
}

template <int D>
struct Tile {
  static constexpr int kG = D / kGroup;                 // groups of a row
  static constexpr int kCodeBytes = 16 * D / 2;         // 16 keys or values
  static constexpr int kScaleBytes = 16 * kG * 2;
  static constexpr int kBytes = 2 * kCodeBytes + 4 * kScaleBytes;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(valid ? N : 0) : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {   // transpose of an 8x8 matrix of 16-bit elements held by the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Codes of nibbles i and 4 + i of a word, minus kMinus, as pair i: (1024 + c) - 1024 - kMinus and (1024 + 16 c) / 16 - 64 - kMinus are
// exact.
template <int kMinus>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&out)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = lop3_and_or(i < 2 ? w : w >> 8, (i & 1) ? 0x00F000F0u : 0x000F000Fu, 0x64006400u);
    __half2 v = *(const __half2*)&u;
    if (i & 1) v = __hfma2(v, __float2half2_rn(0.0625f), __float2half2_rn(-64.f - kMinus));
    else v = __hadd2(v, __float2half2_rn(-1024.f - kMinus));
    out[i] = *(const uint32_t*)&v;
  }
}
// Where 16-byte chunk `ch` of row `r` goes: rows that are read together fall into different banks (K: rows 0..3 at a time,
// V: rows 0, 2, 4, 6 at a time; with D = 128 two rows share 128 bytes, and V keeps a two-way conflict).
template <int D>
__device__ __forceinline__ int k_chunk(int r, int ch) { return ch ^ (D == 256 ? ((r & 3) << 1) : (((r >> 1) & 1) << 1)); }
template <int D>
__device__ __forceinline__ int v_chunk(int r, int ch) { return ch ^ (D == 256 ? (((r >> 1) & 3) << 1) : (((r >> 1) & 1) << 1)); }

template <typename T, int D, int NT, bool kMask>
__global__ void __launch_bounds__((kWarpsOf<D, NT>) * 32, 2) kv4_sdpa_kernel(const SdpaArgs a) {
  constexpr int stages = kStages;
  constexpr int kWarps = (kWarpsOf<D, NT>);
  using TR = MmaTraits<T>;
  using H = MmaTraits<__half>;
  constexpr int G = D / kGroup, CPR = D / 32, KS = D / 16;   // groups, 16-byte chunks of a row's codes, MMA steps of Q K^T
  using TL = Tile<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  uint2* sQ = (uint2*)smem;                                   // [NT][KS][32] fragments of Q^T
  float* sQs = (float*)(smem + NT * KS * 32 * 8);             // [NT][G][8] sums of q over a group
  float* sC = sQs + NT * G * 8;                               // [NT][8] what brings a row's products back to scores
  float* sEv = sC + 8 * NT + warp * 8 * NT;                   // [kWarps][8 NT] exponents that the warp's output rows carry
  constexpr int kFixed = NT * KS * 32 * 8 + NT * (G + 1 + kWarps) * 8 * 4;
  uint8_t* ring = smem + kFixed + warp * stages * TL::kBytes;
  const uint32_t uring = smem_u32(ring);
  pdl_wait();
  pdl_trigger();
  const int split = blockIdx.x, bhk = blockIdx.z, b = bhk / a.Hk, hk = bhk % a.Hk, row0 = blockIdx.y * 8 * NT;
  const int len = a.lengths ? max(a.lengths[b], 0) : a.max_length;
  const int t_last = min(row0 + 8 * NT, a.rows) - 1;
  // one past the last position any row of this block sees
  const int hi = min(min(len, a.max_length), len - a.T + t_last / a.gqa + 1);
  const int tiles = hi > 0 ? (hi + 15) >> 4 : 0;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int tile1 = min(tiles, (split + 1) * per);
  int tile = split * per + warp;

  const uint8_t* kc = (const uint8_t*)(a.k.codes + b * a.k.codes_batch_stride + hk * a.k.codes_head_stride);
  const uint8_t* vc = (const uint8_t*)(a.v.codes + b * a.v.codes_batch_stride + hk * a.v.codes_head_stride);
  const T* ksc = (const T*)a.k.scales + b * a.k.scales_batch_stride + hk * a.k.scales_head_stride;
  const T* kbi = (const T*)a.k.biases + b * a.k.biases_batch_stride + hk * a.k.biases_head_stride;
  const T* vsc = (const T*)a.v.scales + b * a.v.scales_batch_stride + hk * a.v.scales_head_stride;
  const T* vbi = (const T*)a.v.biases + b * a.v.biases_batch_stride + hk * a.v.biases_head_stride;
  // A lane's places: chunk lane % CPR of row lane / CPR + 32 / CPR * i of the codes; key lane & 15 of two of the four scale arrays.
  const uint8_t* kl = kc + lane * 16;
  const uint8_t* vl = vc + lane * 16;
  const T* sl[2] = {((lane & 16) ? kbi : ksc) + (lane & 15) * G, ((lane & 16) ? vbi : vsc) + (lane & 15) * G};
  auto fetch = [&](int tl, int stage) {
    if (tl < tile1) {
      const uint32_t dst = uring + stage * TL::kBytes;
      const int n0 = tl * 16;
      const bool whole = n0 + 16 <= hi;
      const size_t from = (size_t)n0 * (D / 2);
#pragma unroll
      for (int i = 0; i < 16 * CPR / 32; ++i) {
        const int row = lane / CPR + 32 / CPR * i, ch = lane % CPR;
        const bool ok = whole || n0 + row < hi;
        const size_t at = ok ? from + 512 * i : 0;   // 32 chunks of 16 bytes a step
        cp16(dst + row * (D / 2) + k_chunk<D>(row, ch) * 16, kl + at, ok);
        cp16(dst + TL::kCodeBytes + row * (D / 2) + v_chunk<D>(row, ch) * 16, vl + at, ok);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool ok = whole || n0 + (lane & 15) < hi;
        cp_small<2 * G>(dst + 2 * TL::kCodeBytes + (2 * i + (lane >> 4)) * TL::kScaleBytes + (lane & 15) * 2 * G, sl[i] + (ok ? (size_t)n0 * G : 0), ok);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < stages - 1; ++s) fetch(tile + s * kWarps, s);
  if (lane < 8 * NT) sEv[lane] = 0.f;

  // Q^T fragments: a warp per row, a lane per octet j of channels.  In an MMA step lane (r, c) holds row r and the nibble pairs of
  // words 8g + 2c (steps 0 and 1 of group g) and 8g + 2c + 1 (steps 2 and 3).
  for (int row = warp; row < 8 * NT; row += kWarps) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row0 + row < a.rows && lane < D / 8) {
      const int t = (row0 + row) / a.gqa, h = hk * a.gqa + (row0 + row) % a.gqa;
      x = *(const uint4*)((const T*)a.q + b * a.q_sb + h * a.q_sh + t * a.q_st + 8 * lane);
    }
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
    float f[8], big = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = TR::bits_to_float((uint16_t)(u[e >> 1] >> (16 * (e & 1))));
      big = fmaxf(big, fabsf(f[e]));   // NaN is passed over; an infinity makes the row NaN whatever its scale
    }
    const int eq = max((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(big)) >> 23) - 127 - 14, -100);
    const float to_q = __uint_as_float((uint32_t)(127 - eq) << 23);
    float sum = 0.f;
    uint32_t p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 hh = __floats2half2_rn(f[e] * to_q, f[4 + e] * to_q);
      p[e] = *(const uint32_t*)&hh;
      sum += __low2float(hh) + __high2float(hh);
    }
#pragma unroll
    for (int w = 1; w < 8; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    const int nt = row >> 3, rr = row & 7, g = lane >> 3;
    if (lane < D / 8) {
      uint2* dst = sQ + (nt * KS + 4 * g + 2 * (lane & 1)) * 32 + rr * 4 + ((lane & 7) >> 1);
      dst[0] = make_uint2(p[0], p[1]);
      dst[32] = make_uint2(p[2], p[3]);
      if ((lane & 7) == 0) sQs[(nt * G + g) * 8 + rr] = sum;
    }
    if (lane == 0) sC[row] = a.scale * __uint_as_float((uint32_t)(127 + eq) << 23);
  }
  __syncthreads();

  float o[D / 16][NT][4], m[NT][2], l[NT][2], cs[NT][2];
  uint64_t ob[G][NT];   // the rows 2c and 2c + 1 side by side, as in s
  int lim[NT][2];
  long long mat[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[nt][e] = -INFINITY;
      l[nt][e] = 0.f;
      const int row = row0 + nt * 8 + 2 * c + e;
      const int t = row / a.gqa;
      lim[nt][e] = row < a.rows ? min(len - a.T + t, hi - 1) : -1;   // last key the row sees
      mat[nt][e] = kMask && row < a.rows ? b * a.m_sb + (hk * a.gqa + row % a.gqa) * a.m_sh + t * a.m_st : 0;
      cs[nt][e] = sC[nt * 8 + 2 * c + e];
    }
#pragma unroll
    for (int g = 0; g < G; ++g) ob[g][nt] = 0;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
  }
  bool shifted = false;   // whether some row's exponent is not 0

  int stage = 0;
  for (; tile < tile1; tile += kWarps) {
    {
      int ahead = stage + stages - 1;
      if (ahead >= stages) ahead -= stages;
      fetch(tile + (stages - 1) * kWarps, ahead);
    }
    // this tile is the oldest of `stages` groups in flight
    asm volatile("cp.async.wait_group %0;" ::"n"(stages - 1) : "memory");
    __syncwarp();
    const uint8_t* st = ring + stage * TL::kBytes;
    const int n0 = tile * 16;
    // scales of keys r and r + 8
    float sk[2][G], bk[2][G], sv[2][G], bv[2][G];
    float bad[2] = {0.f, 0.f}, big[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint16_t* sc = (const uint16_t*)(st + 2 * TL::kCodeBytes) + (r + 8 * e) * G;
      uint16_t h[4][G];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (G == 4) *(uint2*)h[w] = *(const uint2*)(sc + w * 16 * G);
        else *(uint32_t*)h[w] = *(const uint32_t*)(sc + w * 16 * G);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        sk[e][g] = TR::bits_to_float(h[0][g]);
        bk[e][g] = TR::bits_to_float(h[1][g]);
        sv[e][g] = TR::bits_to_float(h[2][g]);
        const float bb = TR::bits_to_float(h[3][g]);
        bv[e][g] = fmaf(sv[e][g], 8.f, bb);
        bad[e] = fmaf(bv[e][g], 0.f, bad[e]);   // NaN when a scale or bias of the value, or the middle of its codes, is not finite
        big[e] = fmaxf(big[e], fabsf(sv[e][g]));
      }
    }
    if (__any_sync(0xffffffffu, !(bad[0] == 0.f) || !(bad[1] == 0.f))) {
      // keep such a value out of the products (0 * NaN would reach rows that do not see it); rows that do see it get NaN
      // through their scores below
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (!(bad[e] == 0.f)) {
          big[e] = 0.f;
#pragma unroll
          for (int g = 0; g < G; ++g) sv[e][g] = bv[e][g] = 0.f;
        }
    }
    const bool odd = unusual(big[0]) || unusual(big[1]) || shifted;
    bool careful = false;
    // ---- S^T = K Q^T ----
    uint64_t s2[NT][2];   // key r, then r + 8; rows 2c and 2c + 1 side by side
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s2[nt][0] = s2[nt][1] = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint2 w0 = *(const uint2*)(st + r * (D / 2) + k_chunk<D>(r, 2 * g + (c >> 1)) * 16 + (c & 1) * 8);
      const uint2 w1 = *(const uint2*)(st + (r + 8) * (D / 2) + k_chunk<D>(r + 8, 2 * g + (c >> 1)) * 16 + (c & 1) * 8);
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t u0[4], u1[4];
        unpack<0>(half ? w0.y : w0.x, u0);
        unpack<0>(half ? w1.y : w1.x, u1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint2 f = sQ[(nt * KS + 4 * g + 2 * half + ks) * 32 + lane];
            H::mma(acc[nt], u0[2 * ks], u1[2 * ks], u0[2 * ks + 1], u1[2 * ks + 1], f.x, f.y);
          }
      }
      const uint64_t sk0 = pair(sk[0][g], sk[0][g]), sk1 = pair(sk[1][g], sk[1][g]), bk0 = pair(bk[0][g], bk[0][g]), bk1 = pair(bk[1][g], bk[1][g]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint64_t qs = *(const uint64_t*)(sQs + (nt * G + g) * 8 + 2 * c);
        s2[nt][0] = fma2(sk0, pair(acc[nt][0], acc[nt][1]), fma2(bk0, qs, s2[nt][0]));
        s2[nt][1] = fma2(sk1, pair(acc[nt][2], acc[nt][3]), fma2(bk1, qs, s2[nt][1]));
      }
    }
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      unpair(s2[nt][0], s[nt][0], s[nt][1]);
      unpair(s2[nt][1], s[nt][2], s[nt][3]);
    }
    // ---- visibility, running maximum ----
    bool grow = odd;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int n = n0 + r + ((x >> 1) << 3), e = x & 1;
        float t = fmaf(s[nt][x], cs[nt][e], bad[x >> 1]);
        const bool seen = n <= lim[nt][e];
        if (kMask) {
          if (seen) t = apply_mask<T>(a, t, mat[nt][e] + n * a.m_sn);
        }
        t = seen ? t : -INFINITY;
        s[nt][x] = t;
        grow |= t > m[nt][e] + kMaxStep;
      }
    if (__any_sync(0xffffffffu, grow)) {
      // a row's maximum moves for its own scores alone: what other rows see changes no bit of it
      float xk[2] = {0.f, 0.f};   // the keys' own exponents; values of zero ask for none
      bool own[2] = {false, false};
      careful = __any_sync(0xffffffffu, odd);
      if (__builtin_expect(careful, 0)) {
        shifted = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = 0.f, all = 0.f;   // once more: kept, they would cost the usual tiles registers
#pragma unroll
          for (int g = 0; g < G; ++g) {
            top = fmaxf(top, fabsf(sv[e][g]));
            all = fmaxf(all, fmaxf(fabsf(sv[e][g]), fabsf(bv[e][g]) * 0.0625f));
          }
          own[e] = unusual(top);
          if (all == 0.f) xk[e] = -300.f;
          if (own[e]) {
            const int x = max((int)(__float_as_uint(all) >> 23) - 127 - 2, -120);   // 2^(8 - x) |sv| < 2^11
            const float take = __uint_as_float((uint32_t)(127 - x) << 23);
            xk[e] = (float)x;
#pragma unroll
            for (int g = 0; g < G; ++g) { sv[e][g] *= take; bv[e][g] *= take; }
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
          const float before = m[nt][e], now = x > before + kMaxStep ? x : before;
          f[e] = now == -INFINITY ? 1.f : ex2((before - now) * kLog2e);   // nothing seen yet: the sums are zero
          m[nt][e] = now;
          l[nt][e] *= f[e];
          if (__builtin_expect(careful, 0)) {
            float y = fmaxf(fmaf(xk[0], kLn2, s[nt][e]), fmaf(xk[1], kLn2, s[nt][2 + e]));
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, w));
            const float ev = sEv[nt * 8 + 2 * c + e], d = (y - now) * kLog2e;   // octaves of the row's largest p 2^x
            // a row that sees none of the unusual keys, and saw none, stays as it is
            const uint32_t sees = __ballot_sync(0xffffffffu, (own[0] && s[nt][e] != -INFINITY) || (own[1] && s[nt][2 + e] != -INFINITY));
            const bool moves = ((sees >> c) & 0x11111111u) != 0 || ev != 0.f;   // lanes with the same rows
            float ev_now = ev;
            if (moves && now != -INFINITY && (now != before || d > ev + 4.f)) ev_now = fmaxf(ceilf(d), ev + floorf((before - now) * kLog2e));
            if (now != -INFINITY) f[e] = ex2(fmaf(before - now, kLog2e, ev - ev_now));
            __syncwarp();
            if (r == 0) sEv[nt * 8 + 2 * c + e] = ev_now;
            shifted |= ev_now != 0.f;
            // p for the sum, P' without its scale for the products: usual keys under ev = 0 have the same bits in both
            const float ref = now == -INFINITY ? 0.f : now;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float z = s[nt][2 * i + e] - ref;
              l[nt][e] += ex2(z * kLog2e);
              s[nt][2 * i + e] = ex2(fmaf(z, kLog2e, xk[i] - ev_now));
            }
          }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) ob[g][nt] = mul2(ob[g][nt], pair(f[0], f[1]));
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          o[i][nt][0] *= f[0]; o[i][nt][1] *= f[1];
          o[i][nt][2] *= f[0]; o[i][nt][3] *= f[1];
        }
      }
      shifted = __any_sync(0xffffffffu, shifted);
    }
    // ---- p, and O^T += V^T P' per group ----
    if (__builtin_expect(!careful, 1)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float ref = m[nt][x & 1] == -INFINITY ? 0.f : m[nt][x & 1];
          const float p = ex2((s[nt][x] - ref) * kLog2e);
          s[nt][x] = p;
          l[nt][x & 1] += p;
        }
    }
    const uint8_t* sV = st + TL::kCodeBytes;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint32_t pb[NT][2];
      const float s0 = sv[0][g] * kUsual, s1 = sv[1][g] * kUsual;
      const uint64_t bv0 = pair(bv[0][g], bv[0][g]), bv1 = pair(bv[1][g], bv[1][g]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint64_t p0 = pair(s[nt][0], s[nt][1]), p1 = pair(s[nt][2], s[nt][3]);
        float x0, x1, x2, x3;
        unpair(mul2(p0, pair(s0, s0)), x0, x1);
        unpair(mul2(p1, pair(s1, s1)), x2, x3);
        const __half2 h0 = __floats2half2_rn(x0, x1), h1 = __floats2half2_rn(x2, x3);
        pb[nt][0] = movm(*(const uint32_t*)&h0);
        pb[nt][1] = movm(*(const uint32_t*)&h1);
        ob[g][nt] = fma2(p0, bv0, fma2(p1, bv1, ob[g][nt]));
      }
      uint32_t w[4];   // word 8g + r of keys 2c, 2c+1, 2c+8, 2c+9
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * c + (i & 1) + 8 * (i >> 1);
        w[i] = *(const uint32_t*)(sV + key * (D / 2) + v_chunk<D>(key, 2 * g + (r >> 2)) * 16 + (r & 3) * 4);
      }
      // nibbles 0..3 / 4..7 of two keys side by side
      uint32_t lo01[4], hi01[4], lo89[4], hi89[4];
      unpack<8>(prmt(w[0], w[1], 0x5410), lo01);
      unpack<8>(prmt(w[0], w[1], 0x7632), hi01);
      unpack<8>(prmt(w[2], w[3], 0x5410), lo89);
      unpack<8>(prmt(w[2], w[3], 0x7632), hi89);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) H::mma(o[4 * g + t][nt], lo01[t], hi01[t], lo89[t], hi89[t], pb[nt][0], pb[nt][1]);
    }
    if (++stage == stages) stage = 0;
    __syncwarp();   // the buffer is refilled by the next iteration's fetch
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // the rings become the merge buffers

  // ---- merge the warps: O [warp][8 NT][D], m and l [warp][8 NT] ----
  float* mO = (float*)(smem + kFixed);
  float* mM = mO + kWarps * 8 * NT * D;
  float* mL = mM + kWarps * 8 * NT;
  constexpr float undo = 1.f / kUsual;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[nt][e];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
      const int row = nt * 8 + 2 * c + e;
      if (r == 0) {
        mM[warp * 8 * NT + row] = m[nt][e];
        mL[warp * 8 * NT + row] = x;
      }
      float* po = mO + ((size_t)warp * 8 * NT + row) * D;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float y, other;
        if (e == 0) unpair(ob[g][nt], y, other);
        else unpair(ob[g][nt], other, y);
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) y += __shfl_xor_sync(0xffffffffu, y, w);
        float4 v0, v1;   // channels 64g + 8r + 0..3 and + 4..7
        v0.x = fmaf(o[4 * g][nt][e], undo, y); v0.y = fmaf(o[4 * g + 1][nt][e], undo, y);
        v0.z = fmaf(o[4 * g + 2][nt][e], undo, y); v0.w = fmaf(o[4 * g + 3][nt][e], undo, y);
        v1.x = fmaf(o[4 * g][nt][2 + e], undo, y); v1.y = fmaf(o[4 * g + 1][nt][2 + e], undo, y);
        v1.z = fmaf(o[4 * g + 2][nt][2 + e], undo, y); v1.w = fmaf(o[4 * g + 3][nt][2 + e], undo, y);
        *(float4*)(po + 64 * g + 8 * r) = v0;
        *(float4*)(po + 64 * g + 8 * r + 4) = v1;
      }
    }
  __syncthreads();
  const int nrows = min(8 * NT, a.rows - row0);
  for (int i = threadIdx.x; i < nrows * (D / 4); i += kWarps * 32) {
    const int row = i / (D / 4), d = (i % (D / 4)) * 4;
    float mx = -INFINITY, den = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mM[w * 8 * NT + row]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = ex2((mM[w * 8 * NT + row] - ref) * kLog2e);
      den = fmaf(f[w], mL[w * 8 * NT + row], den);
    }
    const float inv = over_sum(den);   // a row that sees nothing yields zeros; NaN stays
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float ev = sC[(1 + w) * 8 * NT + row];   // O carries the row's exponent
      const float fo = (ev == 0.f ? f[w] : ex2(fmaf(mM[w * 8 * NT + row] - ref, kLog2e, ev))) * inv;
      const float4 v = *(const float4*)(mO + ((size_t)w * 8 * NT + row) * D + d);
      acc.x = fmaf(fo, v.x, acc.x); acc.y = fmaf(fo, v.y, acc.y);
      acc.z = fmaf(fo, v.z, acc.z); acc.w = fmaf(fo, v.w, acc.w);
    }
    if (a.splits == 1) {
      const T y[4] = {TR::from_float(acc.x), TR::from_float(acc.y), TR::from_float(acc.z), TR::from_float(acc.w)};
      const float nan = den * 0.f;                       // a NaN sum reaches channels whose own products are finite
      T z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = nan == 0.f ? y[e] : TR::from_float(nan);
      *(uint2*)((T*)a.out + out_row(a, b, hk, row0 + row) * D + d) = *(const uint2*)z;
    } else {
      const size_t at = ((size_t)bhk * a.rows + row0 + row) * a.splits + split;
      *(float4*)(a.part_o + at * D + d) = acc;
      if (d == 0) {
        a.part_m[at] = mx;
        a.part_l[at] = den;
      }
    }
  }
}

constexpr int kMaxSplits = 1024;
// out = sum_s w_s O_s / sum_s w_s, w_s = exp(m_s - max m) l_s: one block per row.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_combine_kernel(const SdpaArgs a) {
  using TR = MmaTraits<T>;
  constexpr int kThreads = 256, kPer = kThreads / (D / 4);   // key ranges read side by side
  __shared__ float sw[kMaxSplits];
  __shared__ float red[kThreads / 32];
  __shared__ float4 part[kPer][D / 4];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row = (size_t)blockIdx.y * a.rows + blockIdx.x;
  const float* pm = a.part_m + row * a.splits;
  const float* pl = a.part_l + row * a.splits;
  const int d4 = tid % (D / 4), s0 = tid / (D / 4);
  const float4* po = (const float4*)(a.part_o + row * a.splits * D) + d4;
  constexpr int kEarly = 8;   // requested before the weights are known
  float4 early[kEarly];
#pragma unroll
  for (int i = 0; i < kEarly; ++i)
    early[i] = s0 + i * kPer < a.splits ? po[(size_t)(s0 + i * kPer) * (D / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
  float mx = -INFINITY;
  for (int s = tid; s < a.splits; s += kThreads) mx = fmaxf(mx, pm[s]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) red[warp] = mx;
  __syncthreads();
  mx = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) mx = fmaxf(mx, red[i]);
  __syncthreads();
  const float ref = mx == -INFINITY ? 0.f : mx;
  float den = 0.f;
  for (int s = tid; s < a.splits; s += kThreads) {
    const float w = ex2((pm[s] - ref) * kLog2e) * pl[s];
    sw[s] = w;
    den += w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  if (lane == 0) red[warp] = den;
  __syncthreads();
  den = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) den += red[i];
  const float inv = over_sum(den), nan = den * 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float w, const float4& v) {
    w *= inv;
    acc.x = fmaf(w, v.x, acc.x); acc.y = fmaf(w, v.y, acc.y);
    acc.z = fmaf(w, v.z, acc.z); acc.w = fmaf(w, v.w, acc.w);
  };
#pragma unroll
  for (int i = 0; i < kEarly; ++i)
    if (s0 + i * kPer < a.splits) add(sw[s0 + i * kPer], early[i]);
#pragma unroll 4
  for (int s = s0 + kEarly * kPer; s < a.splits; s += kPer) add(sw[s], po[(size_t)s * (D / 4)]);
  part[s0][d4] = acc;
  __syncthreads();
  if (s0 != 0) return;
#pragma unroll
  for (int i = 1; i < kPer; ++i) {
    const float4 v = part[i][d4];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  const float v[4] = {acc.x, acc.y, acc.z, acc.w};
  T z[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = TR::from_float(nan == 0.f ? v[e] : nan);
  const int b = blockIdx.y / a.Hk, hk = blockIdx.y % a.Hk;
  *(uint2*)((T*)a.out + out_row(a, b, hk, blockIdx.x) * D + 4 * d4) = *(const uint2*)z;
}

// The same for at most kFewSplits key ranges (many rows, as a prompt has): a thread per four channels of a row, which computes the
// row's weights itself; no block-wide step.
constexpr int kFewSplits = 8;
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_combine_few_kernel(const SdpaArgs a) {
  using TR = MmaTraits<T>;
  pdl_wait();
  pdl_trigger();
  constexpr int kLanes = D / 4;
  const int r = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes, d4 = threadIdx.x % kLanes;
  if (r >= a.rows) return;
  const size_t row = (size_t)blockIdx.y * a.rows + r;
  const float4* po = (const float4*)(a.part_o + row * a.splits * D) + d4;
  float4 v[kFewSplits];
  float m[kFewSplits], l[kFewSplits], mx = -INFINITY;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const bool in = s < a.splits;
    v[s] = in ? po[(size_t)s * kLanes] : make_float4(0.f, 0.f, 0.f, 0.f);
    m[s] = in ? a.part_m[row * a.splits + s] : -INFINITY;
    l[s] = in ? a.part_l[row * a.splits + s] : 0.f;
    mx = fmaxf(mx, m[s]);
  }
  const float ref = mx == -INFINITY ? 0.f : mx;
  float den = 0.f;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    l[s] *= ex2((m[s] - ref) * kLog2e);
    den += l[s];
  }
  const float inv = over_sum(den), nan = den * 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const float w = l[s] * inv;
    acc.x = fmaf(w, v[s].x, acc.x); acc.y = fmaf(w, v[s].y, acc.y);
    acc.z = fmaf(w, v[s].z, acc.z); acc.w = fmaf(w, v[s].w, acc.w);
  }
  const float y[4] = {acc.x, acc.y, acc.z, acc.w};
  T z[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = TR::from_float(nan == 0.f ? y[e] : nan);
  *(uint2*)((T*)a.out + out_row(a, blockIdx.y / a.Hk, blockIdx.y % a.Hk, r) * D + 4 * d4) = *(const uint2*)z;
}

// ---- host side ---------------------------------------------------------------------------------------------------------
int row_tile(int rows) { return rows <= 8 ? 1 : 2; }   // 8-row columns of the MMA tile: 16 query rows share one pass

// Key ranges per (sequence, KV head, row tile), per_sm blocks on an SM at a time.  A block costs its keys and about kOverhead keys'
// worth of start-up and merging.  Equal sequences run in whole waves; sequences of different lengths (several of them: the host
// does not know) fill the SMs as blocks end, behind the longest of which the launch waits: half of each estimate.  (16 sequences of up to
// 32768 keys, 8 rows: lengths drawn evenly 63.8 us against 65.7 by waves alone, equal lengths 82.4 against 78.5; the other sizes tried
// take the same ranges either way.)
constexpr int kOverhead = 320;
int choose_splits(long long units, int B, int max_length, int device, int requested, int per_sm) {
  const int most = (max_length + 127) / 128;
  if (requested > 0) return requested < most ? requested : most;
  const int sms = per_sm * sm_count(device);   // blocks at a time
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= most && s <= kMaxSplits && units * s <= 4ll * sms; ++s) {
    const double keys = (double)max_length / s + kOverhead;
    double cost = (double)((units * s + sms - 1) / sms) * keys;
    if (B > 1) cost = 0.5 * cost + 0.5 * ((double)(units * s) / sms * keys + 0.5 * keys);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

template <typename T, int D, int NT>
int launch_sdpa(SdpaArgs a, cudaStream_t st, int device) {
  constexpr int kWarps = (kWarpsOf<D, NT>);
  using TL = Tile<D>;
  constexpr size_t fixed = (size_t)NT * (D / 16) * 32 * 8 + (size_t)NT * (D / kGroup + 1 + kWarps) * 8 * 4;
  constexpr size_t merge = (size_t)kWarps * 8 * NT * (D + 2) * 4;
  constexpr size_t ring = (size_t)kWarps * kStages * TL::kBytes;
  constexpr size_t smem = fixed + (ring > merge ? ring : merge);
  static_assert(smem <= 113 * 1024, "two blocks of an SM share its memory");
  auto kern = a.mask_kind ? kv4_sdpa_kernel<T, D, NT, true> : kv4_sdpa_kernel<T, D, NT, false>;
  static std::mutex mu;
  static bool done[64][2] = {};
  {
    std::lock_guard<std::mutex> lk(mu);
    bool& d = done[device & 63][a.mask_kind ? 1 : 0];
    if (!d) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return fail(DFLASH_ERR_LAUNCH, "kv4_sdpa: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      d = true;
    }
  }
  const int row_tiles = (a.rows + 8 * NT - 1) / (8 * NT);
  cudaError_t e = launch_kernel(kern, dim3(a.splits, row_tiles, a.B * a.Hk), dim3(kWarps * 32), smem, st, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DFLASH_ERR_LAUNCH, "kv4_sdpa launch: %s", cudaGetErrorString(e));
  return DFLASH_OK;
}

template <typename T, int D>
int launch_combine(const SdpaArgs& a, cudaStream_t st) {
  constexpr int kRowsAtOnce = 256 / (D / 4);
  cudaError_t e = a.splits <= kFewSplits
                      ? launch_kernel(kv4_combine_few_kernel<T, D>, dim3((a.rows + kRowsAtOnce - 1) / kRowsAtOnce, a.B * a.Hk), dim3(256), 0, st, a)
                      : launch_kernel(kv4_combine_kernel<T, D>, dim3(a.rows, a.B * a.Hk), dim3(256), 0, st, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? DFLASH_OK : fail(DFLASH_ERR_LAUNCH, "kv4_sdpa combine launch: %s", cudaGetErrorString(e));
}

template <typename T>
int launch_typed(const SdpaArgs& a, bool tc, int dtype, int D, cudaStream_t st, int device) {
  int rc;
  if (tc) rc = launch_partials_tc(a, dtype, D, st, device);
  else if (row_tile(a.rows) == 1) rc = D == 128 ? launch_sdpa<T, 128, 1>(a, st, device) : launch_sdpa<T, 256, 1>(a, st, device);
  else rc = D == 128 ? launch_sdpa<T, 128, 2>(a, st, device) : launch_sdpa<T, 256, 2>(a, st, device);
  if (rc || a.splits == 1) return rc;
  return D == 128 ? launch_combine<T, 128>(a, st) : launch_combine<T, 256>(a, st);
}

int check_cache(const char* who, const dflash_kv4_cache* c, int D) {
  if (!c || !c->codes || !c->scales || !c->biases) return fail(DFLASH_ERR_BAD_ARG, "%s: null cache array", who);
  const int row = D / kGroup;
  if (((uintptr_t)c->codes & 15) || ((uintptr_t)c->scales & (2 * row - 1)) || ((uintptr_t)c->biases & (2 * row - 1)) ||
      (c->codes_batch_stride & 3) || (c->codes_head_stride & 3) || c->scales_batch_stride % row || c->scales_head_stride % row ||
      c->biases_batch_stride % row || c->biases_head_stride % row)
    return fail(DFLASH_ERR_MISALIGNED, "%s: cache arrays must be aligned to 16 bytes (codes) and to a row (scales, biases)", who);
  return DFLASH_OK;
}

int check_sizes(const char* who, int B, int Hk, int T, int D, int capacity, int dtype) {
  if (B < 0 || Hk < 1 || T < 0) return fail(DFLASH_ERR_BAD_SHAPE, "%s: bad sizes B=%d Hk=%d T=%d", who, B, Hk, T);
  if (D != 128 && D != 256) return fail(DFLASH_ERR_BAD_SHAPE, "%s: D=%d not in {128,256}", who, D);
  if (capacity < 1) return fail(DFLASH_ERR_BAD_SHAPE, "%s: capacity %d", who, capacity);
  if ((long long)B * Hk > 0x7fffffffll) return fail(DFLASH_ERR_BAD_SHAPE, "%s: B*Hk too large", who);
  if (T > 0x7fffffff - (1 << 23)) return fail(DFLASH_ERR_BAD_SHAPE, "%s: T=%d too large", who, T);
  if (dtype != DFLASH_BF16 && dtype != DFLASH_F16) return fail(DFLASH_ERR_BAD_ARG, "%s: dtype %d (want bf16 or f16)", who, dtype);
  return DFLASH_OK;
}

bool aligned_rows(const void* p, const long long* s) {
  return !((uintptr_t)p & 15) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
}

// Steps of a warp: one while the blocks do not fill the SMs (latency), more for long inputs (the next rows' loads in flight).
constexpr int kManyRows = 8;
// Grid of a write or read: (sequence, head) x blocks of rows x sides; true: kManyRows rows a warp.
bool row_grid(int B, int Hk, int T, int D, int sides, int device, dim3* grid) {
  const int per = D == 128 ? 8 : 4;   // rows of a block of four warps, one each
  const long long heads = (long long)B * Hk;
  const bool many = heads * T * sides >= 8ll * per * kManyRows * sm_count(device);
  const long long y = ((long long)T + per * (many ? kManyRows : 1) - 1) / (per * (many ? kManyRows : 1));
  *grid = dim3((unsigned)heads, (unsigned)(y < 65535 ? y : 65535), (unsigned)sides);
  return many;
}

}  // namespace
}  // namespace kv4
}  // namespace dflash

using namespace dflash;
using namespace dflash::kv4;

extern "C" int dflash_kv4_write(const void* keys, const long long* key_strides, const void* values,
                                const long long* value_strides, const dflash_kv4_cache* k_cache,
                                const dflash_kv4_cache* v_cache, const int* offsets, const int* counts, int B, int Hk, int T,
                                int D, int capacity, int dtype, void* stream) {
  int rc = check_sizes("kv4_write", B, Hk, T, D, capacity, dtype);
  if (rc) return rc;
  if (B == 0 || T == 0) return DFLASH_OK;
  if (!keys || !values || !key_strides || !value_strides || !offsets) return fail(DFLASH_ERR_BAD_ARG, "kv4_write: null operand");
  if ((rc = check_cache("kv4_write", k_cache, D)) || (rc = check_cache("kv4_write", v_cache, D))) return rc;
  if (!aligned_rows(keys, key_strides) || !aligned_rows(values, value_strides))
    return fail(DFLASH_ERR_MISALIGNED, "kv4_write: keys and values need 16-byte aligned rows");
  WriteArgs a{};
  a.x[0] = keys; a.x[1] = values;
  for (int i = 0; i < 2; ++i) {
    const long long* s = i ? value_strides : key_strides;
    a.sb[i] = s[0]; a.sh[i] = s[1]; a.st[i] = s[2];
    a.c[i] = i ? *v_cache : *k_cache;
  }
  a.offsets = offsets; a.counts = counts; a.Hk = Hk; a.T = T; a.capacity = capacity;
  int device = 0;
  cudaGetDevice(&device);
  int* err = device_error_word(device);
  if (!err) return fail(DFLASH_ERR_LAUNCH, "kv4_write: no device error word");
  dim3 grid;
  a.steps = row_grid(B, Hk, T, D, 2, device, &grid) ? kManyRows : 1;
  const long long covered = (long long)grid.y * 4 * (D == 128 ? 2 : 1) * a.steps;
  if (covered < T) a.steps = (int)((T + covered / a.steps - 1) / (covered / a.steps));   // grid.y at its limit: longer loops
  const dim3 block(128);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (dtype == DFLASH_BF16)
    e = D == 128 ? launch_kernel(kv4_write_kernel<__nv_bfloat16, 128>, grid, block, 0, st, a, err)
                 : launch_kernel(kv4_write_kernel<__nv_bfloat16, 256>, grid, block, 0, st, a, err);
  else
    e = D == 128 ? launch_kernel(kv4_write_kernel<__half, 128>, grid, block, 0, st, a, err)
                 : launch_kernel(kv4_write_kernel<__half, 256>, grid, block, 0, st, a, err);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? DFLASH_OK : fail(DFLASH_ERR_LAUNCH, "kv4_write launch: %s", cudaGetErrorString(e));
}

extern "C" int dflash_kv4_read(const dflash_kv4_cache* k_cache, const dflash_kv4_cache* v_cache, void* keys_out,
                               void* values_out, const int* starts, int start, int B, int Hk, int T, int D, int capacity,
                               int dtype, void* stream) {
  int rc = check_sizes("kv4_read", B, Hk, T, D, capacity, dtype);
  if (rc) return rc;
  if (B == 0 || T == 0) return DFLASH_OK;
  if (!keys_out) return fail(DFLASH_ERR_BAD_ARG, "kv4_read: null operand");
  if ((rc = check_cache("kv4_read", k_cache, D)) || (values_out && (rc = check_cache("kv4_read", v_cache, D)))) return rc;
  if (((uintptr_t)keys_out & 15) || ((uintptr_t)values_out & 15)) return fail(DFLASH_ERR_MISALIGNED, "kv4_read: outputs must be 16-byte aligned");
  ReadArgs a{};
  a.c[0] = *k_cache;
  if (values_out) a.c[1] = *v_cache;
  a.out[0] = keys_out; a.out[1] = values_out;
  a.starts = starts; a.start = start; a.Hk = Hk; a.T = T; a.capacity = capacity;
  int device = 0;
  cudaGetDevice(&device);
  dim3 grid;
  const bool many = row_grid(B, Hk, T, D, values_out ? 2 : 1, device, &grid);
  const dim3 block(128);
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto one, auto four) { return many ? launch_kernel(four, grid, block, 0, st, a) : launch_kernel(one, grid, block, 0, st, a); };
  cudaError_t e;
  if (dtype == DFLASH_BF16)
    e = D == 128 ? go(kv4_read_kernel<__nv_bfloat16, 128, 1>, kv4_read_kernel<__nv_bfloat16, 128, kManyRows>)
                 : go(kv4_read_kernel<__nv_bfloat16, 256, 1>, kv4_read_kernel<__nv_bfloat16, 256, kManyRows>);
  else
    e = D == 128 ? go(kv4_read_kernel<__half, 128, 1>, kv4_read_kernel<__half, 128, kManyRows>)
                 : go(kv4_read_kernel<__half, 256, 1>, kv4_read_kernel<__half, 256, kManyRows>);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? DFLASH_OK : fail(DFLASH_ERR_LAUNCH, "kv4_read launch: %s", cudaGetErrorString(e));
}

// Whether the rows go to the tcgen05 kernel.  It has the throughput, the other one the shorter way from launch to end: where tiles of 16
// rows fit the SMs side by side and have little to do in all, they are faster (D = 256, 96 rows a KV head, 4 heads: 128 positions 9.8
// against 11.9 us, 512 11.7 against 14.6, 2048 16.4 against 16.3; 4 sequences: 128 positions 10.0 against 12.1, 512 17.3 against 16.2).
static bool takes_tc(int B, int Hk, long long rows, int max_length, int device) {
  if (rows <= kFewRows) return false;
  const long long units = (long long)B * Hk * ((rows + 15) / 16), sms = sm_count(device);
  return units > 2 * sms || units * max_length > 160 * sms;
}
static int kv4_splits(int B, int Hk, long long rows, int max_length, int device, int num_splits) {
  const bool tc = takes_tc(B, Hk, rows, max_length, device);
  const int tile = tc ? kTcRows : 8 * row_tile((int)rows);
  const long long units = (long long)B * Hk * ((rows + tile - 1) / tile);
  return choose_splits(units, B, max_length, device, num_splits, tc ? 1 : 2);
}

extern "C" size_t dflash_kv4_sdpa_workspace_bytes(int B, int Hq, int Hk, int T, int D, int max_length, int num_splits) {
  if (B < 1 || Hq < 1 || Hk < 1 || T < 1 || D < 1 || max_length < 1 || num_splits < 0 || num_splits > kMaxSplits || Hq % Hk != 0 || (long long)(Hq / Hk) * T > 0x7fffffffll) return 0;
  int device = 0;
  cudaGetDevice(&device);
  const long long rows = (long long)(Hq / Hk) * T;
  const int splits = kv4_splits(B, Hk, rows, max_length, device, num_splits);
  return splits > 1 ? (size_t)B * Hk * rows * splits * (D + 2) * sizeof(float) : 0;
}

extern "C" int dflash_kv4_sdpa_plan(int B, int Hq, int Hk, int T, int max_length, int num_splits, int* out, int capacity) {
  if (B < 1 || Hq < 1 || Hk < 1 || Hq % Hk != 0 || T < 1 || max_length < 1 || num_splits < 0 || num_splits > kMaxSplits ||
      (long long)(Hq / Hk) * T > 1000000)
    return fail(DFLASH_ERR_BAD_SHAPE, "kv4_sdpa_plan: bad sizes");
  if (!out || capacity < 2) return fail(DFLASH_ERR_BAD_ARG, "kv4_sdpa_plan: capacity %d < 2", capacity);
  int device = 0;
  cudaGetDevice(&device);
  const long long rows = (long long)(Hq / Hk) * T;
  out[0] = takes_tc(B, Hk, rows, max_length, device);
  out[1] = kv4_splits(B, Hk, rows, max_length, device, num_splits);
  return 2;
}

extern "C" int dflash_kv4_sdpa(const void* q, const long long* q_strides, const dflash_kv4_cache* k_cache,
                               const dflash_kv4_cache* v_cache, const void* mask, int mask_kind, const long long* mask_strides,
                               void* out, const int* lengths, int B, int Hq, int Hk, int T, int D, int capacity, int max_length,
                               float scale, int dtype, int num_splits, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_sizes("kv4_sdpa", B, Hk, T, D, capacity, dtype);
  if (rc) return rc;
  if (Hq < 1 || Hq % Hk != 0) return fail(DFLASH_ERR_BAD_SHAPE, "kv4_sdpa: %d query heads on %d KV heads", Hq, Hk);
  if (!(scale - scale == 0.f)) return fail(DFLASH_ERR_BAD_ARG, "kv4_sdpa: the scale is not finite");
  if (max_length < 0 || max_length > capacity) return fail(DFLASH_ERR_BAD_SHAPE, "kv4_sdpa: max_length %d outside 0..%d", max_length, capacity);
  if (B == 0 || T == 0) return DFLASH_OK;
  if (!q || !q_strides || !out) return fail(DFLASH_ERR_BAD_ARG, "kv4_sdpa: null operand");
  if (mask_kind < 0 || mask_kind > 3 || (mask_kind != 0) != (mask != nullptr) || (mask_kind && !mask_strides))
    return fail(DFLASH_ERR_BAD_ARG, "kv4_sdpa: mask and mask_kind %d do not agree", mask_kind);
  if (num_splits < 0 || num_splits > kMaxSplits) return fail(DFLASH_ERR_BAD_ARG, "kv4_sdpa: num_splits %d outside 0..%d", num_splits, kMaxSplits);
  const int entry = mask_kind == 1 ? 1 : mask_kind == 2 ? 2 : 4;
  if (mask && ((uintptr_t)mask & (entry - 1))) return fail(DFLASH_ERR_MISALIGNED, "kv4_sdpa: a mask must be aligned to its elements");
  if ((rc = check_cache("kv4_sdpa", k_cache, D)) || (rc = check_cache("kv4_sdpa", v_cache, D))) return rc;
  if (!aligned_rows(q, q_strides) || ((uintptr_t)out & 15)) return fail(DFLASH_ERR_MISALIGNED, "kv4_sdpa: q and out need 16-byte aligned rows");
  const long long rows = (long long)(Hq / Hk) * T;
  if ((long long)B * Hk > 65535 || rows > 1000000) return fail(DFLASH_ERR_BAD_SHAPE, "kv4_sdpa: B*Hk=%lld or rows per KV head %lld too large", (long long)B * Hk, rows);
  int device = 0;
  cudaGetDevice(&device);
  SdpaArgs a{};
  a.q = q; a.q_sb = q_strides[0]; a.q_sh = q_strides[1]; a.q_st = q_strides[2];
  a.k = *k_cache; a.v = *v_cache;
  a.mask = mask; a.mask_kind = mask_kind;
  if (mask_kind) { a.m_sb = mask_strides[0]; a.m_sh = mask_strides[1]; a.m_st = mask_strides[2]; a.m_sn = mask_strides[3]; }
  a.out = out; a.lengths = lengths;
  a.B = B; a.Hq = Hq; a.Hk = Hk; a.gqa = Hq / Hk; a.T = T; a.rows = (int)rows;
  a.max_length = max_length; a.scale = scale;
  a.splits = kv4_splits(B, Hk, rows, max_length > 0 ? max_length : 1, device, num_splits);
  if (a.splits > 1) {
    const size_t n = (size_t)B * Hk * rows * a.splits, need = n * (D + 2) * sizeof(float);
    if (!workspace || workspace_bytes < need) return fail(DFLASH_ERR_WORKSPACE, "kv4_sdpa needs %zu workspace bytes, got %zu", need, workspace_bytes);
    if ((uintptr_t)workspace & 15) return fail(DFLASH_ERR_MISALIGNED, "kv4_sdpa workspace must be 16-byte aligned");
    a.part_o = (float*)workspace;
    a.part_m = a.part_o + n * D;
    a.part_l = a.part_m + n;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const bool tc = takes_tc(B, Hk, rows, max_length, device);
  return dtype == DFLASH_BF16 ? launch_typed<__nv_bfloat16>(a, tc, dtype, D, st, device) : launch_typed<__half>(a, tc, dtype, D, st, device);
}
