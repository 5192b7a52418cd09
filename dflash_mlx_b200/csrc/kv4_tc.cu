// Attention over the 4-bit KV cache on the 5th-generation tensor cores, for many query rows per KV head (a verify block of a
// grouped model, a chunk of a prompt); the contract and the formulas are those of kv4.cu.
//
// One block = 128 query rows (row = position * heads-per-KV-head + head, the TMEM lanes of an M128 tile) and a range of keys,
// in tiles of 128: two score tiles and the output fill tensor memory (2 x 128 + 256 columns; narrower score tiles ran at half
// rate, an M128 N64 MMA taking as long as N128).  Keys and values are unpacked to fp16 into 128B-swizzled shared memory: a slab
// per 64 channels (one quantisation group), rows of keys of 128 bytes, which is K-major for S = Q K^T and MN-major for O = P V.
//   warps 0-3   softmax, a thread per row: S from tensor memory, P back over it, O rescaled in place when the maximum moved
//   warps 4-7   unpack keys, 8-11 values: a thread owns a key, a group at a time
//   warp 12     one thread issues the MMAs in the order QK(0) QK(1) PV(0) QK(2) PV(1) ..., so that a tile's softmax runs under
//               the next tile's scores
// One tile of keys and one of values are enough: a slab of keys is free as soon as its four steps of QK(i) are done and is
// refilled under PV(i-1), values (in blocks of 32 keys) the other way round.
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
constexpr int kRows = 128, kKeys = 128;
constexpr int kThreads = 13 * 32, kKeyWarp = 4, kValueWarp = 8, kIssuer = 12;
constexpr float kMaxStep = 8 * kLn2;   // natural units
constexpr float kPShift = 6.f;         // P = p * 2^6 (p <= 2^8): further from fp16's subnormals
constexpr int kSlab = kKeys * 128;     // 128 rows x 64 channels: Q, K or V
constexpr uint32_t kOCol = 256, kCols = 512;   // S / P of tile i at 128 * (i & 1)

// What softmax needs to know about a tile: per 32 keys the power of two of K, the exponent of V, and keys whose value is not
// finite.
struct Meta {
  float k_factor[4];
  int v_exp[4];
  uint32_t bad[4];
};
constexpr int kMeta = 4;   // keys are unpacked at most two tiles ahead of the softmax

// mbarriers, 8 bytes each
enum { kBarKFull = 0, kBarKEmpty = 4, kBarVFull = 8, kBarVEmpty = 12, kBarS = 16, kBarP = 18, kBarO = 20, kBarVMeta = 22, kBarQ = 24, kBars = 26 };

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
// D (+)= A (shared memory descriptor) * B (shared memory descriptor)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)
      : "memory");
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
struct Raw {   // one key: codes, scales and biases of every group
  uint4 c[D / 32];
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
template <bool kWide>
__device__ __forceinline__ void unpack_row(const uint4& c0, const uint4& c1, float scale, float bias, int e, uint32_t row, int key) {
  const float sx = scale * pow2(kWide ? -e : min(24 - e, 127));   // e >= -100
  const uint32_t s0 = splat(sx), s1 = splat(sx * 0.0625f), z = splat(bias * pow2(-e));
  const uint32_t w[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
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

// The keys (kV = false) or values of a block's range, by the four warps of a side: thread = key of the tile.
template <typename T, int D, bool kV>
__device__ __forceinline__ void unpack_side(const dflash_kv4_cache& c, int b, int hk, int k0, int hi, int tiles, uint8_t* buf, uint32_t bar0,
                                            Meta* meta, int* err) {
  constexpr int G = D / kGroup;
  const int w = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, key = w * 32 + lane;
  const uint8_t* codes = (const uint8_t*)(c.codes + b * c.codes_batch_stride + hk * c.codes_head_stride);
  const T* scales = (const T*)c.scales + b * c.scales_batch_stride + hk * c.scales_head_stride;
  const T* biases = (const T*)c.biases + b * c.biases_batch_stride + hk * c.biases_head_stride;
  auto load = [&](int tile, Raw<D>& r) {
    const int n = k0 + tile * kKeys + key;
    if (tile < tiles && n < hi) {
      const uint4* p = (const uint4*)(codes + (size_t)n * (D / 2));
#pragma unroll
      for (int i = 0; i < D / 32; ++i) r.c[i] = __ldg(p + i);
      const T *ps = scales + (size_t)n * G, *pb = biases + (size_t)n * G;
      if (G == 4) {
        const uint2 s = *(const uint2*)ps, z = *(const uint2*)pb;
        r.s[0] = s.x; r.s[G / 2 - 1] = s.y;
        r.b[0] = z.x; r.b[G / 2 - 1] = z.y;
      } else {
        r.s[0] = *(const uint32_t*)ps;
        r.b[0] = *(const uint32_t*)pb;
      }
    } else {   // behind the range: zeros, which no row sees
#pragma unroll
      for (int i = 0; i < D / 32; ++i) r.c[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < D / 128; ++i) r.s[i] = r.b[i] = 0;
    }
  };
  auto done = [&](uint32_t bar) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor pipe reads what was stored
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  Raw<D> cur, next;
  load(0, next);
  bool ok = true;
  for (int t = 0; t < tiles && ok; ++t) {
    cur = next;
    load(t + 1, next);   // in flight under this tile's unpacking and waits
    float s[G], z[G];
    scales_of<T, D>(cur, s, z);
    int e;
    bool wide = false;
    if (kV) wide = wide_range(s, z, &e);
    if (!wide) e = block_exponent(s, z);
    Meta& m = meta[t & (kMeta - 1)];
    if (kV) {
      bool bad = false;
#pragma unroll
      for (int g = 0; g < G; ++g) bad |= !finite(s[g]) || !finite(z[g]);
      if (bad) {   // out of the products; rows that see it get NaN through its score
#pragma unroll
        for (int g = 0; g < G; ++g) s[g] = z[g] = 0.f;
      }
      const uint32_t bads = __ballot_sync(0xffffffffu, bad);
      if (lane == 0) {
        m.v_exp[w] = e;
        m.bad[w] = bads;
        mbar_arrive(bar0 + 8 * (kBarVMeta + (t & 1)));
      }
      // this warp's keys are one block of the values' buffer
      if (!wait_warp(bar0 + 8 * (kBarVEmpty + w), (t & 1) ^ 1)) { atomicCAS(err, 0, 62 | (1 << 8)); ok = false; break; }
    } else if (lane == 0) {
      m.k_factor[w] = pow2(e);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (!kV && !wait_warp(bar0 + 8 * (kBarKEmpty + g), (t & 1) ^ 1)) { atomicCAS(err, 0, 62 | (2 << 8)); ok = false; break; }
      const uint32_t row = smem_u32(buf + g * kSlab + key * 128);
      if (kV && wide) unpack_row<true>(cur.c[2 * g], cur.c[2 * g + 1], s[g], z[g], e, row, key);
      else unpack_row<false>(cur.c[2 * g], cur.c[2 * g + 1], s[g], z[g], e, row, key);
      if (!kV) done(bar0 + 8 * (kBarKFull + g));
    }
    if (kV) done(bar0 + 8 * (kBarVFull + w));
  }
}

template <typename T, int D, bool kMask>
__global__ void __launch_bounds__(kThreads, 1) kv4_sdpa_tc_kernel(const SdpaArgs a, int* __restrict__ err) {
  using TR = MmaTraits<T>;
  constexpr int G = D / kGroup;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + G * kSlab;
  uint8_t* sV = sK + G * kSlab;
  uint64_t* bars = (uint64_t*)(sV + G * kSlab);
  Meta* meta = (Meta*)(bars + kBars);
  int* sE = (int*)(meta + kMeta);                 // exponent of each query row
  uint32_t* holder = (uint32_t*)(sE + kRows);
  const uint32_t bar0 = smem_u32(bars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar0 + 8 * (kBarKFull + i), 4);
      mbar_init(bar0 + 8 * (kBarKEmpty + i), 1);
      mbar_init(bar0 + 8 * (kBarVFull + i), 1);
      mbar_init(bar0 + 8 * (kBarVEmpty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar0 + 8 * (kBarS + i), 1);
      mbar_init(bar0 + 8 * (kBarP + i), 4);
      mbar_init(bar0 + 8 * (kBarO + i), 1);
      mbar_init(bar0 + 8 * (kBarVMeta + i), 4);
    }
    mbar_init(bar0 + 8 * kBarQ, 4);
    mbar_fence_init();
  }
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(kCols) : "memory");
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

  if (warp >= kKeyWarp && warp < kValueWarp) {
    unpack_side<T, D, false>(a.k, b, hk, k0, hi, tiles, sK, bar0, meta, err);
  } else if (warp >= kValueWarp && warp < kIssuer) {
    unpack_side<T, D, true>(a.v, b, hk, k0, hi, tiles, sV, bar0, meta, err);
  } else if (warp == kIssuer) {
    // ---------------- MMA issue ----------------
    if (lane == 0) {
      bool ok = wait_bar(bar0 + 8 * kBarQ, 0);
      if (!ok) atomicCAS(err, 0, 62 | (9 << 8));
      for (int i = 0; i <= tiles && ok && tiles > 0; ++i) {
        if (i < tiles) {   // S(i) = Q K(i)^T
          const uint32_t d = tmem + 128u * (i & 1);
          for (int g = 0; g < G && ok; ++g) {
            if (!wait_bar(bar0 + 8 * (kBarKFull + g), i & 1)) { atomicCAS(err, 0, 62 | (3 << 8)); ok = false; break; }
            fence_after();
            const uint64_t da = desc_k(smem_u32(sQ + g * kSlab)), db = desc_k(smem_u32(sK + g * kSlab));
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_ss(d, da + 2 * j, db + 2 * j, idesc(kKeys, false), (g | j) ? 1u : 0u);
            commit(bar0 + 8 * (kBarKEmpty + g));
          }
          if (!ok) break;
          commit(bar0 + 8 * (kBarS + (i & 1)));
        }
        if (i > 0) {       // O += P(n) V(n); the score tile after next, which takes P(n)'s columns, is issued behind it
          const int n = i - 1;
          if (!wait_bar(bar0 + 8 * (kBarP + (n & 1)), (n >> 1) & 1)) { atomicCAS(err, 0, 62 | (4 << 8)); ok = false; break; }
          for (int blk = 0; blk < 4 && ok; ++blk) {
            if (!wait_bar(bar0 + 8 * (kBarVFull + blk), n & 1)) { atomicCAS(err, 0, 62 | (5 << 8)); ok = false; break; }
            fence_after();
            const uint64_t dv = desc_mn(smem_u32(sV + blk * 32 * 128), kSlab);
#pragma unroll
            for (int j = 0; j < 2; ++j)   // 16 keys = two 1024-byte groups; P: 8 columns (16 fp16)
              mma_ts(tmem + kOCol, tmem + 128u * (n & 1) + 8u * (2 * blk + j), dv + (uint64_t)(j * (2048 >> 4)), idesc(D, true),
                     (n | blk | j) ? 1u : 0u);
            commit(bar0 + 8 * (kBarVEmpty + blk));
          }
          if (!ok) break;
          commit(bar0 + 8 * (kBarO + (n & 1)));
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax: thread = query row ----------------
    const int r = warp * 32 + lane, row = row0 + r;
    const bool row_ok = row < a.rows;
    const bool live = row0 + warp * 32 < a.rows;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int t = row_ok ? row / a.gqa : 0, h = hk * a.gqa + (row_ok ? row % a.gqa : 0);
    // Q: a row per D / 8 lanes, brought to fp16 by a power of two (its largest element to [2^7, 2^8)) in unpack_row's channel order;
    // the scale's sign goes with it, so that scores grow with their products
    {
      constexpr int kLanes = D / 8, kPer = 32 / kLanes, kBatch = 16;
      const int j = lane % kLanes;
#pragma unroll 1
      for (int r0 = warp * 32; r0 < warp * 32 + 32; r0 += kBatch * kPer) {
        uint4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int row = row0 + r0 + i * kPer + lane / kLanes;
          x[i] = make_uint4(0, 0, 0, 0);
          if (row < a.rows) {
            const int t = row / a.gqa, h = hk * a.gqa + row % a.gqa;
            x[i] = *(const uint4*)((const T*)a.q + b * a.q_sb + h * a.q_sh + t * a.q_st + 8 * j);
          }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int r = r0 + i * kPer + lane / kLanes;
          const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          float f[8], big = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = TR::bits_to_float((uint16_t)(u[e >> 1] >> (16 * (e & 1))));
            big = fmaxf(big, finite(f[e]) ? fabsf(f[e]) : 0.f);
          }
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
          const int eq = min(max((int)(__float_as_uint(big) >> 23) - 127 - 7, -100), 126);
          const float to_q = a.scale < 0.f ? -pow2(-eq) : pow2(-eq);
          uint32_t p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 hh = __floats2half2_rn(f[e] * to_q, f[4 + e] * to_q);
            p[e] = *(const uint32_t*)&hh;
          }
          *(uint4*)(sQ + (j >> 3) * kSlab + r * 128 + (((j & 7) ^ (r & 7)) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
          if (j == 0) sE[r] = eq;
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(bar0 + 8 * kBarQ);
    const float c_row = fabsf(a.scale) * pow2(sE[r]);
    // last key the row sees; rows behind the last one compute what nobody reads
    const int lim = row_ok ? min(len - a.T + t, hi - 1) : (kMask ? -1 : 0x7FFFFFFF);
    const long long mat = kMask && row_ok ? b * a.m_sb + h * a.m_sh + t * a.m_st : 0;
    float m = -INFINITY, l = 0.f;
    int ev = -200;   // exponent that O carries
    bool ok = true;
    for (int i = 0; i < tiles; ++i) {
      if (!wait_warp(bar0 + 8 * (kBarS + (i & 1)), (i >> 1) & 1) || !wait_warp(bar0 + 8 * (kBarVMeta + (i & 1)), (i >> 1) & 1)) {
        atomicCAS(err, 0, 62 | (6 << 8));
        ok = false;
        break;
      }
      fence_after();
      if (!live) {   // P is whatever is there: lanes of their own
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar0 + 8 * (kBarP + (i & 1)));
        continue;
      }
      const uint32_t s_col = tmem + lanes + 128u * (i & 1);
      const Meta& mt = meta[i & (kMeta - 1)];
      const int n0 = k0 + i * kKeys;
      const bool plain = !kMask && (mt.bad[0] | mt.bad[1] | mt.bad[2] | mt.bad[3]) == 0 && __all_sync(0xffffffffu, n0 + kKeys - 1 <= lim);
      float top = -INFINITY;
#pragma unroll
      for (int q0 = 0; q0 < 4; q0 += 2) {   // 64 keys at a time
        uint32_t v[64];
        ld32(s_col + 32 * q0, v);
        ld32(s_col + 32 * q0 + 32, v + 32);
        wait_ld();
        if (plain) {
          float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            t0 = fmaxf(t0, __uint_as_float(v[e]));
            t1 = fmaxf(t1, __uint_as_float(v[32 + e]));
          }
          top = fmaxf(top, fmaxf(t0 * (c_row * mt.k_factor[q0]), t1 * (c_row * mt.k_factor[q0 + 1])));
        } else {   // scores as the row sees them, back into their columns
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            const int n = n0 + 32 * q0 + e;
            float x = __uint_as_float(v[e]) * (c_row * mt.k_factor[q0 + (e >> 5)]);
            if ((mt.bad[q0 + (e >> 5)] >> (e & 31)) & 1) x = __int_as_float(0x7FC00000);
            if (n <= lim) {
              if (kMask) x = apply_mask<T>(a, x, mat + n * a.m_sn);
            } else {
              x = -INFINITY;
            }
            top = fmaxf(top, x);
            v[e] = __float_as_uint(x);
          }
#pragma unroll
          for (int e = 0; e < 64; e += 16) st16(s_col + 32 * q0 + e, v + e);
          wait_st();
        }
      }
      const int ev_tile = max(max(mt.v_exp[0], mt.v_exp[1]), max(mt.v_exp[2], mt.v_exp[3]));
      if (__any_sync(0xffffffffu, top > m + kMaxStep) || ev_tile > ev) {
        const float m_new = fmaxf(m, top);
        const int ev_new = max(ev, ev_tile);
        const float f = m_new == -INFINITY ? 1.f : ex2((m - m_new) * kLog2e);
        const float fo = f * pow2(max(ev - ev_new, -126));
        l *= f;
        m = m_new;
        if (i > 0) {
          if (!wait_warp(bar0 + 8 * (kBarO + ((i - 1) & 1)), ((i - 1) >> 1) & 1)) { atomicCAS(err, 0, 62 | (7 << 8)); ok = false; break; }
          fence_after();
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            ld32(tmem + lanes + kOCol + c0, o);
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fo);
            st16(tmem + lanes + kOCol + c0, o);
            st16(tmem + lanes + kOCol + c0 + 16, o + 16);
          }
          wait_st();
        }
        ev = ev_new;
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t v[32];
        ld32(s_col + 32 * q, v);
        wait_ld();
        const float shift = kPShift + (float)max(mt.v_exp[q] - ev, -100);   // P carries V's power of two
        const float cl = plain ? c_row * mt.k_factor[q] * kLog2e : kLog2e, off = shift - ref * kLog2e;
        float sum0 = 0.f, sum1 = 0.f;
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float x0 = __uint_as_float(v[e]), x1 = __uint_as_float(v[e + 1]);
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
        st16(s_col + 16 * q, w);   // over columns that have been read
      }
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar0 + 8 * (kBarP + (i & 1)));
    }
    // ---- epilogue: the row goes through shared memory (all of Q, K and V is spent), so that it leaves as one bulk copy ----
    // the last product; the one two before it is done (its successor's scores were), so the phase cannot be mistaken
    if (tiles > 0 && ok && !wait_warp(bar0 + 8 * (kBarO + ((tiles - 1) & 1)), ((tiles - 1) >> 1) & 1)) { atomicCAS(err, 0, 62 | (8 << 8)); ok = false; }
    fence_after();
    const bool have = tiles > 0 && ok;
    if (live) {
      const float undo = pow2(min(max(ev - (int)kPShift, -126), 127));
      const bool last = a.splits == 1;
      const float inv = l == 0.f ? 1.f : 1.f / l, nan = l * 0.f;   // a row that sees nothing yields zeros; NaN reaches the whole row
      const size_t at = ((size_t)bhk * a.rows + row) * a.splits + split;
      uint8_t* stage = smem + r * (D * 4 + 16);   // rows 16 bytes apart modulo 128: no bank conflicts
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t o[32];
        if (have) {
          ld32(tmem + lanes + kOCol + c0, o);
          wait_ld();
        }
        float y[32];   // back to the channels' order
#pragma unroll
        for (int e = 0; e < 32; ++e) y[(e & ~7) + ((e & 1) << 2) + ((e & 7) >> 1)] = have ? __uint_as_float(o[e]) * undo : 0.f;
        if (last) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            T z[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) z[x] = TR::from_float(nan == 0.f ? y[e + x] * inv : nan);
            *(uint4*)(stage + (c0 + e) * 2) = *(const uint4*)z;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *(float4*)(stage + (c0 + e) * 4) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (row_ok) {
        const void* dst = last ? (const void*)((T*)a.out + out_row(a, b, hk, row) * D) : (const void*)(a.part_o + at * D);
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(stage)), "r"(last ? D * 2 : D * 4)
                     : "memory");
        if (!last) {
          a.part_m[at] = m;
          a.part_l[at] = l;
        }
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kIssuer)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

template <typename T, int D>
int launch(const SdpaArgs& a, cudaStream_t st, int device) {
  constexpr size_t tiles = (size_t)3 * (D / kGroup) * kSlab, rest = kBars * 8 + kMeta * sizeof(Meta) + kRows * 4 + 16;
  static_assert(kRows * (D * 4 + 16) <= tiles, "the epilogue's rows fit where Q, K and V were");
  constexpr size_t smem = tiles + rest;
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
  cudaError_t e = launch_kernel(kern, grid, dim3(kThreads), smem, st, a, err);
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
