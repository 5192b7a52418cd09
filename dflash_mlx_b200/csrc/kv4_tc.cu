// Attention over the 4-bit KV cache on the 5th-generation tensor cores, for many query rows per KV head (a verify block of a
// grouped model, a chunk of a prompt); the contract and the formulas are those of kv4.cu.
//
// One block = 128 query rows (row = position * heads-per-KV-head + head, the TMEM lanes of an M128 tile) and a range of keys,
// in tiles of 64.  Keys and values are unpacked to fp16 into 128B-swizzled shared memory, a ring of buffers that alternate
// K(0) V(0) K(1) V(1) ...; both have rows of keys with 64 channels (one quantisation group) each 128 bytes, which is K-major for
// S = Q K^T and MN-major for O = P V.
//   warps 0-3  softmax, a thread per row: S from tensor memory, P back over it, O rescaled in place when the maximum moved
//   next 2 * (D/64) warps unpack: a thread owns the 64 channels of one key and group, i.e. one scale and one 128-byte row
//   last warp  one thread issues the MMAs in the order QK(0) QK(1) PV(0) QK(2) PV(1) ..., so that a tile's softmax runs under
//              the next tile's scores
// Q sits in tensor memory too (A operand of QK), so that the tensor pipe reads only K and V from shared memory.
//
// Unpacking costs 9 instructions for 8 codes: a nibble left in place is an fp16 subnormal, code * 2^-24 (or * 2^-20), and one packed
// fma turns two of them into code * scale + bias with a single rounding to fp16 (2^-11; the cache's scales carry 8 or 11 bits,
// the codes 4).  For that, every 32 keys share a power of two that brings the scales under 2^-8 and that S (for K) or P (for V)
// takes back.  Values far below the largest of their 32 keys lose bits at 2^-21 of that largest one: nothing to a score, and values
// of keys that differ by more than 6 octaves are unpacked in 13 instructions with 16 more bits of range.  q is brought
// to fp16 by a power of two per row, exact down to 2^-22 of the row's largest element.  P is fp16, up to 2^14.
// The running maximum moves only when a score exceeds it by 8 octaves.  Every wait is bounded (device error code 62).
#include <mutex>

#include "kv4.cuh"

namespace dflash {
namespace kv4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRows = 128, kKeys = 64;
constexpr float kMaxStep = 8 * kLn2;   // natural units
constexpr float kPShift = 6.f;         // P = p * 2^6 (p <= 2^8): further from fp16's subnormals

template <int D>
struct Shape {
  static constexpr int kG = D / kGroup;
  static constexpr int kUnpackWarps = 2 * kG;
  static constexpr int kThreads = (4 + kUnpackWarps + 1) * 32;
  static constexpr int kSlots = D == 256 ? 6 : 8;
  static constexpr int kSlab = kKeys * 128;            // 64 keys x 64 channels
  static constexpr int kBuf = kG * kSlab;
  static constexpr uint32_t kQCol = 0, kSCol = D / 2, kOCol = 256, kCols = 512;
};

// What softmax needs to know about a tile: per 32 keys the power of two of K, the exponent of V, and keys whose value is not
// finite.
struct Meta {
  float k_factor[2];
  int v_exp[2];
  uint32_t bad[2];
};
constexpr int kMeta = 8;   // tiles in flight are at most 4

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 16); ++i) {   // hardware-suspended polls of up to a microsecond
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(1000u)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// The same for a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_bar(bar, parity)); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D (+)= A (tensor memory) * B (shared memory descriptor)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// K-major operand, 128B swizzle: rows of 128 bytes (64 channels), 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// MN-major operand, 128B swizzle: a row is one k index holding 64 consecutive n, 8 k = one 1024-byte group, the next 64 n lie
// `lbo` bytes further.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// kind::f16 instruction descriptor: D = f32, A = B = f16, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

template <int D>
struct Raw {   // one key's codes of one group, and its scales and biases of every group
  uint4 c0, c1;
  uint32_t s[D / 128], b[D / 128];
};

template <typename T, int D>
__device__ __forceinline__ void scales_of(const Raw<D>& r, float (&s)[D / kGroup], float (&b)[D / kGroup]) {
#pragma unroll
  for (int g = 0; g < D / kGroup; ++g) {
    s[g] = MmaTraits<T>::bits_to_float((uint16_t)(r.s[g >> 1] >> (16 * (g & 1))));
    b[g] = MmaTraits<T>::bits_to_float((uint16_t)(r.b[g >> 1] >> (16 * (g & 1))));
  }
}
// Exponent e shared by the warp's 32 keys: scale * 2^-e < 2^-9 and |bias| * 2^-e < 2^14 for the finite ones.
template <int G>
__device__ __forceinline__ int block_exponent(const float (&s)[G], const float (&b)[G]) {
  float ms = 0.f, mb = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    ms = fmaxf(ms, finite(s[g]) ? fabsf(s[g]) : 0.f);
    mb = fmaxf(mb, finite(b[g]) ? fabsf(b[g]) : 0.f);
  }
  const int es = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(ms)) >> 23) - 127;
  const int eb = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(mb)) >> 23) - 127;
  return min(max(max(es + 10, eb - 13), -100), 126);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t splat(float x) {
  const __half2 h = __float2half2_rn(x);
  return *(const uint32_t*)&h;
}
// Exponent for unpack_row's wide form: |scale| * 15 + |bias| of every finite key is below 2^14 after it, and whether the keys
// are too unlike for the narrow form: a key's largest value is more than 6 octaves below the largest of the 32.
template <int G>
__device__ __forceinline__ bool wide_range(const float (&s)[G], const float (&b)[G], int* e) {
  float mine = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float x = fmaf(fabsf(s[g]), 15.f, fabsf(b[g]));
    mine = fmaxf(mine, finite(x) ? x : 0.f);
  }
  const uint32_t u = __float_as_uint(mine) >> 23;
  const int hi = (int)__reduce_max_sync(0xffffffffu, u), lo = (int)__reduce_min_sync(0xffffffffu, mine == 0.f ? 255u : u);
  *e = min(max(hi - 127 - 13, -100), 126);
  return hi - lo > 6 && lo < 255;
}
// 64 codes -> a swizzled 128-byte row; the eight codes of a word land in the order 0 4 1 5 2 6 3 7.  Narrow: the nibbles are
// fp16 subnormals and one fma makes the value (9 instructions a word); wide: the nibbles become whole numbers first (13).
template <int D, bool kWide>
__device__ __forceinline__ void unpack_row(const Raw<D>& r, float scale, float bias, int e, uint32_t row, int key) {
  const float sx = scale * pow2(kWide ? -e : min(24 - e, 127));   // e >= -100
  const uint32_t s0 = splat(sx), s1 = splat(sx * 0.0625f), z = splat(bias * pow2(-e));
  const uint32_t w[8] = {r.c0.x, r.c0.y, r.c0.z, r.c0.w, r.c1.x, r.c1.y, r.c1.z, r.c1.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = j < 2 ? w[i] : w[i] >> 8;
      if (kWide) {
        const uint32_t u = lop3_and_or(x, (j & 1) ? 0x00F000F0u : 0x000F000Fu, 0x64006400u);
        // 1024 + c -> c and 1024 + 16 c -> c, exactly
        const uint32_t c = (j & 1) ? hfma2(u, 0x2C002C00u, 0xD400D400u) : hfma2(u, 0x3C003C00u, 0xE400E400u);
        v[j] = hfma2(c, s0, z);
      } else {
        v[j] = hfma2(x & ((j & 1) ? 0x00F000F0u : 0x000F000Fu), (j & 1) ? s1 : s0, z);
      }
    }
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(row + ((uint32_t)(i ^ (key & 7)) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3])
                 : "memory");
  }
}

template <typename T, int D, bool kMask>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1) kv4_sdpa_tc_kernel(const SdpaArgs a, int* __restrict__ err) {
  using S = Shape<D>;
  using TR = MmaTraits<T>;
  constexpr int G = S::kG;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  uint64_t* bars = (uint64_t*)(smem + S::kSlots * S::kBuf);
  Meta* meta = (Meta*)(bars + 2 * S::kSlots + 8);
  uint32_t* holder = (uint32_t*)(meta + kMeta);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * S::kSlots, bar_q = bar_empty + 8 * S::kSlots;
  const uint32_t bar_s = bar_q + 8, bar_p = bar_s + 16, bar_o = bar_p + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kIssuer = 4 + S::kUnpackWarps;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(bar_full + 8 * i, S::kUnpackWarps);
      mbar_init(bar_empty + 8 * i, 1);
    }
    mbar_init(bar_q, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_s + 8 * i, 1);
      mbar_init(bar_p + 8 * i, 4);
      mbar_init(bar_o + 8 * i, 1);
    }
    mbar_fence_init();
  }
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(S::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *holder;
  pdl_wait();
  pdl_trigger();
  const int split = blockIdx.x, bhk = blockIdx.z, b = bhk / a.Hk, hk = bhk % a.Hk, row0 = blockIdx.y * kRows;
  const int len = a.lengths ? a.lengths[b] : a.max_length;
  const int t_last = (min(row0 + kRows, a.rows) - 1) / a.gqa;
  // one past the last position any row of this block sees
  const int hi = min(min(len, a.max_length), len - a.T + t_last + 1);
  const int tiles_all = hi > 0 ? (hi + kKeys - 1) / kKeys : 0;
  const int per = (tiles_all + a.splits - 1) / a.splits;
  const int k0 = split * per * kKeys;
  const int tiles = max(0, min(tiles_all - split * per, per));

  if (warp >= 4 && warp < kIssuer) {
    // ---------------- unpack ----------------
    const int dw = warp - 4, half = dw & 1, g = dw >> 1, key = half * 32 + lane;
    const dflash_kv4_cache* sides[2] = {&a.k, &a.v};
    const uint8_t* codes[2];
    const T *scales[2], *biases[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      codes[v] = (const uint8_t*)(sides[v]->codes + b * sides[v]->codes_batch_stride + hk * sides[v]->codes_head_stride) + 32 * g;
      scales[v] = (const T*)sides[v]->scales + b * sides[v]->scales_batch_stride + hk * sides[v]->scales_head_stride;
      biases[v] = (const T*)sides[v]->biases + b * sides[v]->biases_batch_stride + hk * sides[v]->biases_head_stride;
    }
    auto load = [&](int tile, int v, Raw<D>& r) {
      const int n = k0 + tile * kKeys + key;
      if (tile < tiles && n < hi) {
        const uint4* p = (const uint4*)(codes[v] + (size_t)n * (D / 2));
        r.c0 = __ldg(p);
        r.c1 = __ldg(p + 1);
        const T *ps = scales[v] + (size_t)n * G, *pb = biases[v] + (size_t)n * G;
        if (G == 4) {
          const uint2 s = *(const uint2*)ps, z = *(const uint2*)pb;
          r.s[0] = s.x; r.s[G / 2 - 1] = s.y;
          r.b[0] = z.x; r.b[G / 2 - 1] = z.y;
        } else {
          r.s[0] = *(const uint32_t*)ps;
          r.b[0] = *(const uint32_t*)pb;
        }
      } else {   // behind the range: zeros, which no row sees
        r.c0 = r.c1 = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < D / 128; ++i) r.s[i] = r.b[i] = 0;
      }
    };
    constexpr int kAhead = 2;   // tiles in registers: about a memory latency of unpacking
    Raw<D> rk[kAhead], rv[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      load(i, 0, rk[i]);
      load(i, 1, rv[i]);
    }
    bool ok = true;
    int slot = 0;
    uint32_t phase = 1;   // the first pass over the ring does not wait
    for (int t0 = 0; t0 < tiles && ok; t0 += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int t = t0 + u;
        if (t < tiles && ok) {
          float s[G], z[G], sv[G], zv[G];
          scales_of<T, D>(rk[u], s, z);
          scales_of<T, D>(rv[u], sv, zv);
          const int ek = block_exponent(s, z);
          int ev;
          const bool wide = wide_range(sv, zv, &ev);
          if (!wide) ev = block_exponent(sv, zv);
          bool bad = false;
#pragma unroll
          for (int i = 0; i < G; ++i) bad |= !finite(sv[i]) || !finite(zv[i]);
          const uint32_t bads = __ballot_sync(0xffffffffu, bad);
          if (g == 0 && lane == 0) {
            Meta& m = meta[t & (kMeta - 1)];
            m.k_factor[half] = pow2(ek);
            m.v_exp[half] = ev;
            m.bad[half] = bads;
          }
          float mine_s = s[0], mine_z = z[0], mine_sv = sv[0], mine_zv = zv[0];
#pragma unroll
          for (int i = 1; i < G; ++i)
            if (i == g) { mine_s = s[i]; mine_z = z[i]; mine_sv = sv[i]; mine_zv = zv[i]; }
          if (bad) mine_sv = mine_zv = 0.f;   // out of the products; rows that see it get NaN through its score
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            if (!wait_warp(bar_empty + 8 * slot, phase)) { atomicCAS(err, 0, 62 | (1 << 8)); ok = false; break; }
            const uint32_t row = smem_u32(ring + slot * S::kBuf + g * S::kSlab + key * 128);
            if (v == 0) {
              unpack_row<D, false>(rk[u], mine_s, mine_z, ek, row, key);
              load(t + kAhead, 0, rk[u]);
            } else {
              if (wide) unpack_row<D, true>(rv[u], mine_sv, mine_zv, ev, row, key);
              else unpack_row<D, false>(rv[u], mine_sv, mine_zv, ev, row, key);
              load(t + kAhead, 1, rv[u]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor pipe reads what was stored
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_full + 8 * slot);
            if (++slot == S::kSlots) { slot = 0; phase ^= 1; }
          }
        }
      }
    }
  } else if (warp == kIssuer) {
    // ---------------- MMA issue ----------------
    if (lane == 0 && tiles > 0) {
      bool ok = wait_bar(bar_q, 0);
      if (!ok) atomicCAS(err, 0, 62 | (2 << 8));
      fence_after();
      for (int i = 0; i <= tiles && ok; ++i) {
        if (i < tiles) {   // S(i) = Q K(i)^T
          const int seq = 2 * i, slot = seq % S::kSlots;
          if (!wait_bar(bar_full + 8 * slot, (seq / S::kSlots) & 1)) { atomicCAS(err, 0, 62 | (3 << 8)); ok = false; break; }
          fence_after();
          const uint32_t d = tmem + S::kSCol + 64u * (i & 1);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            mma_ts(d, tmem + S::kQCol + 8u * ks, desc_k(smem_u32(ring + slot * S::kBuf + (ks >> 2) * S::kSlab)) + 2 * (ks & 3),
                   idesc(kKeys, false), ks ? 1u : 0u);
          commit(bar_empty + 8 * slot);
          commit(bar_s + 8 * (i & 1));
        }
        if (i > 0) {       // O += P(j) V(j)
          const int j = i - 1, seq = 2 * j + 1, slot = seq % S::kSlots;
          if (!wait_bar(bar_p + 8 * (j & 1), (j >> 1) & 1)) { atomicCAS(err, 0, 62 | (4 << 8)); ok = false; break; }
          if (!wait_bar(bar_full + 8 * slot, (seq / S::kSlots) & 1)) { atomicCAS(err, 0, 62 | (5 << 8)); ok = false; break; }
          fence_after();
          const uint64_t dv = desc_mn(smem_u32(ring + slot * S::kBuf), S::kSlab);
#pragma unroll
          for (int ks = 0; ks < kKeys / 16; ++ks)   // 16 keys = two 1024-byte groups; P: 8 columns (16 fp16)
            mma_ts(tmem + S::kOCol, tmem + S::kSCol + 64u * (j & 1) + 8u * ks, dv + (uint64_t)(ks * (2048 >> 4)), idesc(D, true),
                   (j | ks) ? 1u : 0u);
          commit(bar_empty + 8 * slot);
          commit(bar_o + 8 * (j & 1));
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax: thread = query row ----------------
    const int row = row0 + warp * 32 + lane;
    const bool row_ok = row < a.rows;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int t = row_ok ? row / a.gqa : 0, h = hk * a.gqa + (row_ok ? row % a.gqa : 0);
    // Q: the row's largest exponent, then fp16 in the channel order of unpack_row
    const uint4* q = (const uint4*)((const T*)a.q + b * a.q_sb + h * a.q_sh + t * a.q_st);
    float big = 0.f;
    for (int i = 0; i < D / 8; ++i) {
      const uint4 x = row_ok ? q[i] : make_uint4(0, 0, 0, 0);
      const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = TR::bits_to_float((uint16_t)(u[e >> 1] >> (16 * (e & 1))));
        big = fmaxf(big, finite(f) ? fabsf(f) : 0.f);
      }
    }
    const int eq = min(max((int)(__float_as_uint(big) >> 23) - 127 - 7, -100), 126);   // largest element in [2^7, 2^8)
    const float to_q = a.scale < 0.f ? -pow2(-eq) : pow2(-eq);   // the scale's sign goes with q: scores then grow with their products
    for (int i0 = 0; i0 < D / 8; i0 += 4) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 x = row_ok ? q[i0 + i] : make_uint4(0, 0, 0, 0);
        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = TR::bits_to_float((uint16_t)(u[e >> 1] >> (16 * (e & 1)))) * to_q;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __half2 p = __floats2half2_rn(f[e], f[4 + e]);
          w[4 * i + e] = *(const uint32_t*)&p;
        }
      }
      st16(tmem + lanes + S::kQCol + 4 * i0, w);
    }
    wait_st();
    fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_q);

    const float c_row = fabsf(a.scale) * pow2(eq);
    // last key the row sees; rows behind the last one compute what nobody reads
    const int lim = row_ok ? min(len - a.T + t, hi - 1) : (kMask ? -1 : 0x7FFFFFFF);
    const bool live = row0 + warp * 32 < a.rows;
    const long long mat = kMask && row_ok ? b * a.m_sb + h * a.m_sh + t * a.m_st : 0;
    float m = -INFINITY, l = 0.f;
    int ev = -200;   // exponent that O carries
    bool ok = true;
    for (int i = 0; i < tiles; ++i) {
      if (!wait_warp(bar_s + 8 * (i & 1), (i >> 1) & 1)) { atomicCAS(err, 0, 62 | (6 << 8)); ok = false; break; }
      fence_after();
      if (!live) {   // P is whatever is there: lanes of their own
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + 8 * (i & 1));
        continue;
      }
      const uint32_t s_col = tmem + lanes + S::kSCol + 64u * (i & 1);
      uint32_t v[64];
      ld32(s_col, v);
      ld32(s_col + 32, v + 32);
      const Meta mt = meta[i & (kMeta - 1)];
      const int n0 = k0 + i * kKeys;
      wait_ld();
      float c[2] = {c_row * mt.k_factor[0], c_row * mt.k_factor[1]};
      const bool plain = !kMask && (mt.bad[0] | mt.bad[1]) == 0 && __all_sync(0xffffffffu, n0 + kKeys - 1 <= lim);
      float top = -INFINITY;
      if (plain) {
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          t0 = fmaxf(t0, __uint_as_float(v[e]));
          t1 = fmaxf(t1, __uint_as_float(v[32 + e]));
        }
        top = fmaxf(t0 * c[0], t1 * c[1]);
      } else {
#pragma unroll
        for (int e = 0; e < 64; ++e) {
          const int n = n0 + e;
          float x = __uint_as_float(v[e]) * c[e >> 5];
          if ((mt.bad[e >> 5] >> (e & 31)) & 1) x = __int_as_float(0x7FC00000);
          if (n <= lim) {
            if (kMask) x = apply_mask<T>(a, x, mat + n * a.m_sn);
          } else {
            x = -INFINITY;
          }
          top = fmaxf(top, x);
          v[e] = __float_as_uint(x);
        }
        c[0] = c[1] = 1.f;
      }
      const int ev_tile = max(mt.v_exp[0], mt.v_exp[1]);
      if (__any_sync(0xffffffffu, top > m + kMaxStep) || ev_tile > ev) {
        const float m_new = fmaxf(m, top);
        const int ev_new = max(ev, ev_tile);
        const float f = m_new == -INFINITY ? 1.f : ex2((m - m_new) * kLog2e);
        const float fo = f * pow2(max(ev - ev_new, -126));
        l *= f;
        m = m_new;
        if (i > 0) {
          if (!wait_warp(bar_o + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1)) { atomicCAS(err, 0, 62 | (7 << 8)); ok = false; break; }
          fence_after();
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            ld32(tmem + lanes + S::kOCol + c0, o);
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fo);
            st16(tmem + lanes + S::kOCol + c0, o);
            st16(tmem + lanes + S::kOCol + c0 + 16, o + 16);
          }
          wait_st();
        }
        ev = ev_new;
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const float shift = kPShift + (float)max(mt.v_exp[hf] - ev, -100);   // P carries V's power of two
        const float cl = c[hf] * kLog2e, off = shift - ref * kLog2e;
        float sum0 = 0.f, sum1 = 0.f;
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float x0 = __uint_as_float(v[32 * hf + e]), x1 = __uint_as_float(v[32 * hf + e + 1]);
          float p0, p1;
          if (kMask) {   // scores may be the lowest finite value: their difference first
            p0 = ex2(fmaf(x0 - ref, kLog2e, shift));
            p1 = ex2(fmaf(x1 - ref, kLog2e, shift));
          } else {
            p0 = ex2(fmaf(x0, cl, off));
            p1 = ex2(fmaf(x1, cl, off));
          }
          sum0 += p0;
          sum1 += p1;
          const __half2 p = __floats2half2_rn(p0, p1);
          w[e >> 1] = *(const uint32_t*)&p;
        }
        l = fmaf(sum0 + sum1, ex2(-shift), l);
        st16(s_col + 16 * hf, w);   // over scores that are in registers
      }
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p + 8 * (i & 1));
    }
    // ---- epilogue ----
    // the last product; the one two before it is done (its successor's scores were), so the phase cannot be mistaken
    if (tiles > 0 && ok && !wait_warp(bar_o + 8 * ((tiles - 1) & 1), ((tiles - 1) >> 1) & 1)) { atomicCAS(err, 0, 62 | (8 << 8)); ok = false; }
    fence_after();
    const bool have = tiles > 0 && ok;
    const float undo = pow2(min(max(ev - (int)kPShift, -126), 127));
    const bool last = a.splits == 1;
    const float inv = l == 0.f ? 1.f : 1.f / l, nan = l * 0.f;   // a row that sees nothing yields zeros; NaN reaches the whole row
    const size_t at = ((size_t)bhk * a.rows + row) * a.splits + split;
    for (int c0 = 0; c0 < D; c0 += 32) {
      uint32_t o[32];
      if (have) {
        ld32(tmem + lanes + S::kOCol + c0, o);
        wait_ld();
      }
      float y[32];   // back to the channels' order
#pragma unroll
      for (int e = 0; e < 32; ++e) y[(e & ~7) + ((e & 1) << 2) + ((e & 7) >> 1)] = have ? __uint_as_float(o[e]) * undo : 0.f;
      if (row_ok) {
        if (last) {
          T* dst = (T*)a.out + out_row(a, b, hk, row) * D + c0;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            T z[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) z[x] = TR::from_float(nan == 0.f ? y[e + x] * inv : nan);
            *(uint4*)(dst + e) = *(const uint4*)z;
          }
        } else {
          float4* dst = (float4*)(a.part_o + at * D + c0);
#pragma unroll
          for (int e = 0; e < 32; e += 4) dst[e >> 2] = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
        }
      }
    }
    if (row_ok && !last) {
      a.part_m[at] = m;
      a.part_l[at] = l;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kIssuer)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kCols) : "memory");
}

template <typename T, int D>
int launch(const SdpaArgs& a, cudaStream_t st, int device) {
  using S = Shape<D>;
  constexpr size_t smem = (size_t)S::kSlots * S::kBuf + (2 * S::kSlots + 8) * 8 + kMeta * sizeof(Meta) + 16;
  static_assert(smem <= 227 * 1024, "shared memory");
  auto kern = a.mask_kind ? kv4_sdpa_tc_kernel<T, D, true> : kv4_sdpa_tc_kernel<T, D, false>;
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
  int* err = device_error_word(device);
  if (!err) return fail(DFLASH_ERR_LAUNCH, "kv4_sdpa: no device error word");
  const dim3 grid(a.splits, (a.rows + kRows - 1) / kRows, a.B * a.Hk);
  cudaError_t e = launch_kernel(kern, grid, dim3(S::kThreads), smem, st, a, err);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? DFLASH_OK : fail(DFLASH_ERR_LAUNCH, "kv4_sdpa (tcgen05) launch: %s", cudaGetErrorString(e));
}

}  // namespace

int launch_partials_tc(const SdpaArgs& a, int dtype, int D, cudaStream_t st, int device) {
  if (dtype == DFLASH_BF16) return D == 128 ? launch<__nv_bfloat16, 128>(a, st, device) : launch<__nv_bfloat16, 256>(a, st, device);
  return D == 128 ? launch<__half, 128>(a, st, device) : launch<__half, 256>(a, st, device);
}

}  // namespace kv4
}  // namespace dflash
