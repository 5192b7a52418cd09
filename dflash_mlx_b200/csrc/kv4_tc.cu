// Attention over the 4-bit KV cache on the 5th-generation tensor cores, for many query rows per KV head (a verify block of a
// grouped model, a chunk of a prompt); the contract and the formulas are those of kv4.cu.
//
// One block = 128 query rows (row = position * heads-per-KV-head + head, the TMEM lanes of an M128 tile) and a range of keys,
// in pairs of 64-key tiles: two pairs of score tiles and the output fill tensor memory (2 x 128 + 256 columns).  Keys and values are
// unpacked to fp16 into 128B-swizzled shared memory: a slab per 64 channels (one quantisation group), rows of keys of 128 bytes,
// which is K-major for S = Q K^T and MN-major for O = P V.  Scores are multiplied by pairs (an M128 N64 MMA takes 55 clocks, N128 64),
// softmax and output go tile by tile.
//   warps 0-7    softmax, a thread per row: S from tensor memory, P back over it, O rescaled in place when the maximum moved.  Warps
//                0-3 take the even tiles and 4-7 the odd ones; a row's reference maximum is handed from one to the other right
//                after a tile's maxima
//   warps 8-11   unpack keys, 12-15 values: a thread owns a key, a group at a time
//   warp 16      one thread issues S = Q K^T, warp 17 O += P V: issuing an MMA blocks until the pipe has room and a satisfied wait
//                costs about 100 cycles of it, so each thread waits under the other one's MMAs
// A slab of keys is refilled as soon as its steps are done, either half of the values while the other one is multiplied.
//
// Unpacking costs 13 instructions for 8 codes: nibbles become whole numbers, and one packed fma makes two of them code * scale + bias
// with a single rounding to fp16 (at most 2^-11 of a value, 2^-25 of the unit below; the cache's scales carry 8 or 11 bits, the codes 4).
// A row must not notice keys that it does not see, so nothing is shared between keys: a key or value whose largest element lies in
// [2^-10, 2^11) is multiplied by 2^4 like all of its kind; any other one by a power of two of its own, which brings that
// element into [2^14, 2^15), so that its other elements are kept to 2^-39 of it.  A column of S takes the power back before its softmax, and P for V: P = p 2^(6 + x - ev), with an
// exponent ev of the row's output that is 0 until the row sees such a value.  Tiles without them, under rows with ev = 0, do not
// touch any of this, and the bits of usual keys are the same either way.  (An exponent shared by 32 keys allows 9 instructions for 8
// codes, 3 % of a long range, but then one large key, seen or not, takes the others' bits.  A cache of unusual keys takes 1.4 times as
// long, one of unusual values 1.6 to 1.8 times.)  q is brought to fp16 by a power of two per row, exact
// down to 2^-22 of the row's largest element.  P is fp16, up to 2^15; its sum takes the unrounded p.
// The running maximum moves only when a score exceeds it by 8 octaves, per row.  Every wait is bounded (device error code 62).
//
// Measured (D = 256, bf16): 128 rows x 131072 keys on 2 KV heads 52 us with the combine: 58 clocks a key and SM at 1.965 GHz, start and end
// included.  No unit is full: issue slots 50 %, shared memory's load / store pipe 42 %, tensor pipe 32 %, HBM 23 %; warps wait for
// one another's tiles.  96 rows x 8192 keys on 4 heads: 20.4 us.
#include <mutex>
#include <type_traits>

#include "kv4.cuh"

namespace dflash {
namespace kv4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kUnit = -4, kUsualFrom = -10, kUsualTo = 11;   // usual keys and values: in units of 2^kUnit, their largest element's octaves
constexpr int kRows = 128, kKeys = 128, kTile = 64;   // keys are unpacked by 128, multiplied by 64
constexpr int kThreads = 18 * 32, kKeyWarp = 8, kValueWarp = 12, kIssuer = 16;   // kIssuer: scores; the next warp: output
constexpr float kPShift = 6.f;         // P = p * 2^6 (p <= 2^9): further from fp16's subnormals
constexpr int kSlab = kKeys * 128;     // 128 rows x 64 channels: Q, K or V
constexpr uint32_t kOCol = 256, kCols = 512;   // S / P of tile i at 64 * (i & 3)

// What softmax needs to know about 128 keys, a bit of a word per key: keys and values that are unusual or not finite, values that are
// not finite; and the exponents of blocks of 32 keys or values with an odd one.
struct __align__(16) Meta {
  int8_t k_exp[128], v_exp[128];
  uint32_t k_odd[4], v_odd[4], v_bad[4];
};
constexpr int kOdd = 1024;               // on a query row's exponent: an element is not finite
constexpr int kMeta = 4;   // scales are looked at no more than three tiles ahead of the softmax

// mbarriers, 8 bytes each.  kBarKEmpty: per slab; V full and empty: per half of the buffer (64 keys); kBarS: per pair of score tiles;
// P, O: per tile in flight; kBarM: a row reference handed on, per tile parity and 32 rows; kBarVMeta: the values' part of Meta of
// 128 keys is known
enum { kBarKFull = 0, kBarQ = 1, kBarVFull = 2, kBarKEmpty = 4, kBarVEmpty = 8, kBarS = 10, kBarP = 12, kBarO = 16, kBarM = 20,
       kBarVMeta = 28, kBars = 32 };

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
// D (+)= A (shared memory descriptor) * B (shared memory descriptor); descriptors as their two halves, of which a step through
// shared memory changes the lower one only
template <bool kAccum>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %6, 0;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(kAccum ? 1 : 0)
      : "memory");
}
// D (+)= A (tensor memory) * B (shared memory descriptor)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accum)
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
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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

// Scales (or biases) of one key from their packed pairs.
template <typename T, int D>
__device__ __forceinline__ void scales_of(const uint32_t (&r)[D / 128], float (&s)[D / kGroup]) {
#pragma unroll
  for (int g = 0; g < D / kGroup; ++g) s[g] = MmaTraits<T>::bits_to_float((uint16_t)(r[g >> 1] >> (16 * (g & 1))));
}
// The largest element a key may hold, as bits: that of codes 0 and 15 over its groups; not finite where one of them is not.
template <int G>
__device__ __forceinline__ uint32_t largest_bits(const float (&s)[G], const float (&b)[G]) {
  uint32_t m = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) m = max(max(m, __float_as_uint(b[g]) & 0x7FFFFFFFu), __float_as_uint(fmaf(s[g], 15.f, b[g])) & 0x7FFFFFFFu);
  return m;
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
// kWords words of a mask row from byte `from` on, whatever its alignment: aligned 16-byte loads, all in flight at once, then shifted
// into place (3 instructions a word).  A lane's row is its own, so narrower loads would cost a line of the L1 each.  Words from `end`
// on are 0.  What an aligned word holds besides bytes of the row (never used) lies in the row's allocation too; a branch for
// it would make the loads wait for one another.
template <int kWords>
__device__ __forceinline__ void mask_words(const uint8_t* row, long long from, long long end, bool want, uint32_t (&w)[kWords + 4]) {
  const uint8_t* p = row + from;
  const int s = (int)((uintptr_t)p & 15);
  const int left = want ? (int)min(end - from + s, (long long)(4 * kWords + 16)) : 0;   // bytes of the row from the first aligned word on
#pragma unroll
  for (int i = 0; i <= kWords; i += 4) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (4 * i < left && (i < kWords || s != 0)) x = *(const uint4*)(p - s + 4 * i);
    w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
  }
#pragma unroll
  for (int i = 0; i < kWords + 2; ++i) w[i] = (s & 8) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < kWords + 1; ++i) w[i] = (s & 4) ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (s & 3));
}
// Bit e of word q: the byte mask's entry of key n0 + 32 q + e is not 0, for the keys up to `lim` (from `end` on none is read).
// `shared`: the warp's rows have one mask row, which its lanes read together.
__device__ __forceinline__ void mask_bits(const SdpaArgs& a, long long mat, bool shared, int n0, int lim, int end, uint32_t (&bits)[2]) {
  const uint8_t* row = (const uint8_t*)a.mask + mat;
  bits[0] = bits[1] = 0;
  if (shared) {
    const int n = n0 + (threadIdx.x & 31);
    const uint8_t x0 = n < end ? row[n * a.m_sn] : 0, x1 = n + 32 < end ? row[(n + 32) * a.m_sn] : 0;
    bits[0] = __ballot_sync(0xffffffffu, x0 != 0);
    bits[1] = __ballot_sync(0xffffffffu, x1 != 0);
  } else if (a.m_sn == 1) {
    uint32_t w[kTile / 4 + 4], zero = 0;
    mask_words<kTile / 4>(row, n0, a.max_length, lim >= n0, w);
#pragma unroll
    for (int i = 0; i < kTile / 4; ++i) zero |= (w[i] - 0x01010101u) & ~w[i];
    if (__all_sync(0xffffffffu, (zero & 0x80808080u) == 0)) {   // no zero byte anywhere
      bits[0] = bits[1] = 0xFFFFFFFFu;
    } else {
#pragma unroll
      for (int i = 0; i < kTile / 4; ++i) {
        const uint32_t x = __vcmpne4(w[i], 0) & 0x08040201u;   // a bit of its own per byte
        bits[i >> 3] |= (((x * 0x01010101u) >> 24) & 15u) << (4 * (i & 7));
      }
    }
  } else {
#pragma unroll 8
    for (int e = 0; e < kTile; ++e)
      if (n0 + e <= lim && row[(n0 + e) * a.m_sn] != 0) bits[e >> 5] |= 1u << (e & 31);
  }
}
// Entries of keys n0 .. of an additive mask of type E as they lie in memory, as many as fit kWords; behind `lim` anything.
template <typename E, int kWords>
__device__ __forceinline__ void mask_entries(const SdpaArgs& a, long long mat, int n0, int lim, uint32_t (&w)[kWords + 4]) {
  constexpr int kPer = 4 / (int)sizeof(E);
  const E* row = (const E*)a.mask + mat;
  if (a.m_sn == 1) {
    mask_words<kWords>((const uint8_t*)row, (long long)n0 * sizeof(E), (long long)a.max_length * sizeof(E), lim >= n0, w);
  } else {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int n = n0 + i * kPer + e;
        if (n > lim) continue;
        if (sizeof(E) == 4) w[i] = ((const uint32_t*)row)[n * a.m_sn];
        else w[i] |= (uint32_t)((const uint16_t*)row)[n * a.m_sn] << (16 * e);
      }
    }
  }
}
// Keys n0 .. n0 + 31 that a row sees, without a mask: up to `lim`.
__device__ __forceinline__ uint32_t seen_bits(int n0, int lim) {
  const int left = lim - n0;   // below 0: none, from 31: all
  return left < 0 ? 0u : left >= 31 ? 0xFFFFFFFFu : (2u << left) - 1u;
}
// Per half, the larger magnitude of two pairs (the sign bits are to be ignored).
template <typename T> __device__ __forceinline__ uint32_t abs_max(uint32_t x, uint32_t y);
template <> __device__ __forceinline__ uint32_t abs_max<__nv_bfloat16>(uint32_t x, uint32_t y) {
  x &= 0x7FFF7FFFu; y &= 0x7FFF7FFFu;
  const __nv_bfloat162 m = __hmax2(*(const __nv_bfloat162*)&x, *(const __nv_bfloat162*)&y);
  return *(const uint32_t*)&m;
}
template <> __device__ __forceinline__ uint32_t abs_max<__half>(uint32_t x, uint32_t y) {
  x &= 0x7FFF7FFFu; y &= 0x7FFF7FFFu;
  const __half2 m = __hmax2(*(const __half2*)&x, *(const __half2*)&y);
  return *(const uint32_t*)&m;
}
// 64 codes -> a swizzled 128-byte row of code * scale + bias (both in the key's unit); the eight codes of a word land in the order
// 0 4 1 5 2 6 3 7.
__device__ __forceinline__ void unpack_row(const uint4& c0, const uint4& c1, float scale, float bias, uint32_t row, int key) {
  const uint32_t s = splat(scale), z = splat(bias);
  const uint32_t w[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = lop3_and_or(j < 2 ? w[i] : w[i] >> 8, (j & 1) ? 0x00F000F0u : 0x000F000Fu, 0x64006400u);
      // 1024 + c -> c and 1024 + 16 c -> c, exactly
      const uint32_t c = (j & 1) ? hfma2(u, 0x2C002C00u, 0xD400D400u) : hfma2(u, 0x3C003C00u, 0xE400E400u);
      v[j] = hfma2(c, s, z);
    }
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(row + ((uint32_t)(i ^ (key & 7)) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3])
                 : "memory");
  }
}

// What takes a key's own power of two back (1 for usual ones), and the exponents of sixteen values; blocks of 32 without an odd one
// have stale exponents.
__device__ __forceinline__ float own_power(const Meta& m, int key) { return m.k_odd[key >> 5] ? pow2(m.k_exp[key]) : 1.f; }
__device__ __forceinline__ uint4 own_exponents(const Meta& m, int key) {
  return m.v_odd[key >> 5] ? *(const uint4*)(m.v_exp + key) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ float exponent(const uint4& x, int e) {
  return (float)(int8_t)(((e >> 2) == 0 ? x.x : (e >> 2) == 1 ? x.y : (e >> 2) == 2 ? x.z : x.w) >> (8 * (e & 3)));
}

// The order in which a block works through its keys: from the last ones back, 64 at a time, so that under masks that fall with the
// distance the largest scores come first and O is not rescaled with every tile (64 rows x 4 x 5001 keys of 256 channels: 40.2 -> 34.1
// us).  A last pair of tiles that is no more than half full comes last, so that its empty half costs nothing.
struct Order {
  int k0, last;    // first key of the range; number of the last pair that goes backwards
  __device__ __forceinline__ int base(int pair) const { return k0 + kKeys * (pair > last ? pair : last - pair); }   // first key of a pair
  __device__ __forceinline__ int flip(int pair) const { return pair > last ? 0 : kTile; }                           // its key in place i: i ^ flip
};
// The keys (kV = false) or values of a block's range, by the four warps of a side: thread = key of the tile.
template <int D>
__device__ __forceinline__ int raw_chunk(int r, int ch) { return D == 256 ? ch ^ (r & 7) : ch ^ ((r >> 1) & 3); }
template <typename T, int D, bool kV, typename F>
__device__ __forceinline__ void unpack_side(const dflash_kv4_cache& c, int b, int hk, const Order& order, int hi, int tiles, uint8_t* buf, uint8_t* raw,
                                            uint32_t bar0, Meta* meta, int* err, F query_rows) {
  constexpr int G = D / kGroup;
  const int w = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, key = w * 32 + lane;
  const uint8_t* codes = (const uint8_t*)(c.codes + b * c.codes_batch_stride + hk * c.codes_head_stride);
  const T* scales = (const T*)c.scales + b * c.scales_batch_stride + hk * c.scales_head_stride;
  const T* biases = (const T*)c.biases + b * c.biases_batch_stride + hk * c.biases_head_stride;
  constexpr int kChunks = D / 32, kRowsAtOnce = 32 / kChunks;   // 16-byte chunks of a key, keys of one load
  raw += w * 32 * (D / 2);
  const uint32_t uraw = smem_u32(raw);
  // This warp's 32 keys of a tile: codes by coalesced asynchronous copies (a lane loading its own key's row would touch 32 lines
  // with every instruction, which measured as the kernel's bound), swizzled so that a lane then reads its row without bank
  // conflicts; scales and biases to registers.  Behind the range: zeros, which no row sees.
  auto load = [&](int tile) {
    const int n0 = order.base(tile) + (w * 32 ^ order.flip(tile));
    const bool in = tile < tiles;
    if (in) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int r = i * kRowsAtOnce + lane / kChunks, ch = lane % kChunks;
        const bool ok = n0 + r < hi;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(uraw + r * (D / 2) + raw_chunk<D>(r, ch) * 16),
                     "l"(codes + (size_t)(ok ? n0 + r : 0) * (D / 2) + ch * 16), "r"(ok ? 16 : 0)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto load_scales = [&](int tile, uint32_t (&s)[D / 128], uint32_t (&z)[D / 128]) {
    const int n = order.base(tile) + (key ^ order.flip(tile));
#pragma unroll
    for (int i = 0; i < D / 128; ++i) s[i] = z[i] = 0;
    if (tile < tiles && n < hi) {
      const T *ps = scales + (size_t)n * G, *pb = biases + (size_t)n * G;
      if (G == 4) {
        const uint2 x = *(const uint2*)ps, y = *(const uint2*)pb;
        s[0] = x.x; s[G / 2 - 1] = x.y;
        z[0] = y.x; z[G / 2 - 1] = y.y;
      } else {
        s[0] = *(const uint32_t*)ps;
        z[0] = *(const uint32_t*)pb;
      }
    }
  };
  auto done = [&](uint32_t bar) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor pipe reads what was stored
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  // Scales of a tile, a tile ahead of its codes: what the values' say about the tile is published before the codes' buffer is free.
  uint32_t ns[D / 128], nz[D / 128];
  float s[G], z[G];   // in the key's unit
  auto prepare = [&](int tile) {
    scales_of<T, D>(ns, s);
    scales_of<T, D>(nz, z);
    const uint32_t largest = largest_bits(s, z);
    const bool bad = largest >= 0x7F800000u;
    const bool usual = largest - ((uint32_t)(127 + kUsualFrom) << 23) < ((uint32_t)(kUsualTo - kUsualFrom) << 23) || largest == 0;
    float unit = pow2(-kUnit);
    const uint32_t odd = __ballot_sync(0xffffffffu, !usual);
    Meta& m = meta[tile & (kMeta - 1)];
    if (odd != 0) {
      int x = 0;
      if (kV && largest == 0) x = -128;   // a value of zero asks for no exponent
      if (!usual && !bad) {   // 2^(kUnit + x): the largest element to [2^14, 2^15)
        x = max((int)(largest >> 23) - 127 - 14 - kUnit, -120);
        unit = pow2(-kUnit - x);
      }
      if (kV && bad) {        // out of the products; rows that see it get NaN through its score
#pragma unroll
        for (int g = 0; g < G; ++g) s[g] = z[g] = 0.f;
      }
      if (tile < tiles) (kV ? m.v_exp : m.k_exp)[key] = (int8_t)x;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) { s[g] *= unit; z[g] *= unit; }
    if (kV) {
      const uint32_t bads = __ballot_sync(0xffffffffu, bad);
      if (lane == 0 && tile < tiles) {
        m.v_odd[w] = odd;
        m.v_bad[w] = bads;
        mbar_arrive(bar0 + 8 * (kBarVMeta + (tile & (kMeta - 1))));
      }
    } else if (lane == 0 && tile < tiles) {
      m.k_odd[w] = odd;
    }
  };
  // the block's queries are converted while the first keys and values are on their way
  load(0);
  load_scales(0, ns, nz);
  asm volatile("cp.async.wait_group 1;" ::: "memory");
  query_rows();
  prepare(0);
  load_scales(1, ns, nz);
  for (int t = 0; t < tiles; ++t) {
    float cs[G], cz[G];
#pragma unroll
    for (int g = 0; g < G; ++g) { cs[g] = s[g]; cz[g] = z[g]; }
    if (kV) {
      prepare(t + 1);
      load_scales(t + 2, ns, nz);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    // two warps share a half of the values' buffer
    if (kV && !wait_warp(bar0 + 8 * (kBarVEmpty + (w >> 1)), (t & 1) ^ 1)) { atomicCAS(err, 0, 62 | (1 << 8)); break; }
    bool ok = true;
#pragma unroll 1
    for (int g = 0; g < G; ++g) {
      if (!kV && !wait_warp(bar0 + 8 * (kBarKEmpty + g), (t & 1) ^ 1)) { atomicCAS(err, 0, 62 | (2 << 8)); ok = false; break; }
      const uint4 c0 = *(const uint4*)(raw + lane * (D / 2) + raw_chunk<D>(lane, 2 * g) * 16);
      const uint4 c1 = *(const uint4*)(raw + lane * (D / 2) + raw_chunk<D>(lane, 2 * g + 1) * 16);
      float sg = cs[0], zg = cz[0];
#pragma unroll
      for (int i = 1; i < G; ++i)
        if (i == g) { sg = cs[i]; zg = cz[i]; }
      const uint32_t row = smem_u32(buf + g * kSlab + key * 128);
      unpack_row(c0, c1, sg, zg, row, key);
    }
    if (!ok) break;
    done(bar0 + 8 * (kV ? kBarVFull + (w >> 1) : kBarKFull));
    load(t + 1);
    if (!kV) {   // a tile's exponents are published with its codes: nothing waits for them before
      prepare(t + 1);
      load_scales(t + 2, ns, nz);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, int D, int kMask>   // 0 = no mask, 1 = bytes, 2 = additive in T, 3 = additive in fp32
__global__ void __launch_bounds__(kThreads, 1) kv4_sdpa_tc_kernel(const SdpaArgs a, int* __restrict__ err) {
  using TR = MmaTraits<T>;
  constexpr int G = D / kGroup;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + G * kSlab;
  uint8_t* sV = sK + G * kSlab;
  uint8_t* sRaw = sV + G * kSlab;                 // codes of the next tile: keys, then values
  uint64_t* bars = (uint64_t*)(sRaw + kKeys * D);
  Meta* meta = (Meta*)(bars + kBars);
  float* sRef = (float*)(meta + kMeta);           // reference maximum of a row, handed from tile to tile
  int16_t* sE = (int16_t*)(sRef + kRows);     // exponent of each query row, + kOdd if the row is not finite
  int8_t* sEv = (int8_t*)(sE + kRows);            // exponent that a row of O carries
  int* sOwn = (int*)(sEv + kRows);                // [4] whether some row of 32 carries one that is not 0
  uint32_t* holder = (uint32_t*)(sOwn + 4);
  float2* sEnd = (float2*)sRaw;                   // [2][128] reference and sum of either half of the softmax, at the end
  const uint32_t bar0 = smem_u32(bars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(bar0 + 8 * kBarKFull, 4);
    mbar_init(bar0 + 8 * kBarQ, kIssuer);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar0 + 8 * (kBarVFull + i), 2);
      mbar_init(bar0 + 8 * (kBarVEmpty + i), 1);
      mbar_init(bar0 + 8 * (kBarS + i), 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar0 + 8 * (kBarKEmpty + i), 1);
      mbar_init(bar0 + 8 * (kBarP + i), 4);
      mbar_init(bar0 + 8 * (kBarO + i), 1);
      mbar_init(bar0 + 8 * (kBarVMeta + i), 4);
    }
    for (int i = 0; i < 8; ++i) mbar_init(bar0 + 8 * (kBarM + i), 1);
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
  // Q: a row per D / 8 lanes, brought to fp16 by a power of two (its largest element to [2^7, 2^8)) in unpack_row's channel order;
  // the scale's sign goes with it, so that scores grow with their products.  Sixteen warps, every sixteenth row each.
  constexpr int kLanes = D / 8, kPer = 32 / kLanes, kSteps = kRows / (kIssuer * kPer);
  auto query_copy = [&]() {   // raw into place, all copies in flight at once
    const int j = lane % kLanes;
#pragma unroll 2
    for (int i = 0; i < kSteps; ++i) {
      const int r = (i * kIssuer + warp) * kPer + lane / kLanes, row = row0 + r;
      const bool in = row < a.rows;
      const int t = in ? row / a.gqa : 0, h = hk * a.gqa + (in ? row - t * a.gqa : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(sQ + (j >> 3) * kSlab + r * 128 + (((j & 7) ^ (r & 7)) << 4))),
                   "l"((const T*)a.q + b * a.q_sb + h * a.q_sh + t * a.q_st + 8 * j), "r"(in ? 16 : 0)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (warp < kIssuer) query_copy();   // the length, which everything below needs, is on its way meanwhile
  const int len = a.lengths ? max(a.lengths[b], 0) : a.max_length;
  const int t_last = (min(row0 + kRows, a.rows) - 1) / a.gqa;
  // one past the last position any row of this block sees
  const int hi = min(min(len, a.max_length), len - a.T + t_last + 1);
  const int tiles_all = hi > 0 ? (hi + kKeys - 1) / kKeys : 0;
  const int per = (tiles_all + a.splits - 1) / a.splits;
  const int k0 = split * per * kKeys;
  const int pairs = max(0, min(tiles_all - split * per, per));                    // 128 keys each
  const bool half = pairs > 0 && hi - k0 <= pairs * kKeys - kTile;                // the last pair's second tile is empty
  const int tiles = 2 * pairs - half;                                             // 64 keys each
  const Order order{k0, pairs - 1 - half};
  auto query_rows = [&]() {   // once they have landed; a lane reads what it copied itself
    const int j = lane % kLanes;
#pragma unroll 2
    for (int i = 0; i < kSteps; ++i) {
      const int r = (i * kIssuer + warp) * kPer + lane / kLanes;
      uint4* place = (uint4*)(sQ + (j >> 3) * kSlab + r * 128 + (((j & 7) ^ (r & 7)) << 4));
      const uint4 x = *place;
      const uint32_t u[4] = {x.x, x.y, x.z, x.w};
      // largest magnitude of the row, NaN passed over (an infinity makes the row NaN whatever its scale)
      uint32_t top = abs_max<T>(abs_max<T>(u[0], u[1]), abs_max<T>(u[2], u[3]));
      top = __float_as_uint(fmaxf(TR::bits_to_float((uint16_t)(top & 0x7FFFu)), TR::bits_to_float((uint16_t)((top >> 16) & 0x7FFFu))));
      if (kLanes == 32) {
        top = __reduce_max_sync(0xffffffffu, top);
      } else {
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      const int eq = min(max((int)(top >> 23) - 127 - 7, -100), 126);
      const float to_q = a.scale < 0.f ? -pow2(-eq) : pow2(-eq);
      uint32_t p[4];
      float odd = 0.f;   // NaN if an element is not finite
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f0 = TR::bits_to_float((uint16_t)(u[e >> 1] >> (16 * (e & 1)))), f1 = TR::bits_to_float((uint16_t)(u[2 + (e >> 1)] >> (16 * (e & 1))));
        const __half2 hh = __floats2half2_rn(f0 * to_q, f1 * to_q);
        if (kMask >= 2) odd = fmaf(f0, 0.f, fmaf(f1, 0.f, odd));
        p[e] = *(const uint32_t*)&hh;
      }
      *place = make_uint4(p[0], p[1], p[2], p[3]);
      const bool is_odd = kMask >= 2 && (__ballot_sync(0xffffffffu, odd != 0.f) >> (lane & ~(kLanes - 1)) & (0xFFFFFFFFu >> (32 - kLanes))) != 0;
      if (j == 0) sE[r] = (int16_t)(is_odd ? eq + kOdd : eq);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(bar0 + 8 * kBarQ);
  };

  if (warp >= kKeyWarp && warp < kValueWarp) {
    unpack_side<T, D, false>(a.k, b, hk, order, hi, pairs, sK, sRaw, bar0, meta, err, query_rows);
  } else if (warp >= kValueWarp && warp < kIssuer) {
    unpack_side<T, D, true>(a.v, b, hk, order, hi, pairs, sV, sRaw + kKeys * D / 2, bar0, meta, err, query_rows);
  } else if (warp == kIssuer) {
    // ---------------- scores ----------------
    if (lane == 0) {
      bool ok = wait_bar(bar0 + 8 * kBarQ, 0);
      if (!ok) atomicCAS(err, 0, 62 | (9 << 8));
      const uint32_t da = (uint32_t)desc_k(smem_u32(sQ)), db = (uint32_t)desc_k(smem_u32(sK)), hi32 = (uint32_t)(desc_k(0) >> 32);
      for (int i = 0; i < pairs && ok; ++i) {
        // the columns hold P of the pair before last until its products are done (both halves: it was not the last pair)
        if (i >= 2 && !wait_bar(bar0 + 8 * (kBarO + ((2 * i - 3) & 3)), ((2 * i - 3) >> 2) & 1)) { atomicCAS(err, 0, 62 | (11 << 8)); break; }
        if (!wait_bar(bar0 + 8 * kBarKFull, i & 1)) { atomicCAS(err, 0, 62 | (3 << 8)); break; }
        fence_after();
        const uint32_t d = tmem + 128u * (i & 1);
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t step = g * (kSlab >> 4) + 2 * j;
            if ((g | j) == 0) mma_ss<false>(d, da, hi32, db, hi32, idesc(kKeys, false));
            else mma_ss<true>(d, da + step, hi32, db + step, hi32, idesc(kKeys, false));
          }
          commit(bar0 + 8 * (kBarKEmpty + g));
        }
        commit(bar0 + 8 * (kBarS + (i & 1)));
      }
    }
    __syncwarp();
  } else if (warp == kIssuer + 1) {
    // ---------------- output ----------------
    if (lane == 0) {
      const uint32_t dv = (uint32_t)desc_mn(smem_u32(sV), kSlab), hi32 = (uint32_t)(desc_mn(0, 0) >> 32);
      for (int i = 0; i < tiles; ++i) {
        if (!wait_bar(bar0 + 8 * (kBarVFull + (i & 1)), (i >> 1) & 1)) { atomicCAS(err, 0, 62 | (5 << 8)); break; }
        if (!wait_bar(bar0 + 8 * (kBarP + (i & 3)), (i >> 2) & 1)) { atomicCAS(err, 0, 62 | (4 << 8)); break; }
        fence_after();
        const uint32_t pc = tmem + 64u * (i & 3), dh = dv + (i & 1) * (kTile * 128 >> 4);
#pragma unroll
        for (int j = 0; j < kTile / 16; ++j)   // 16 keys = two 1024-byte groups; P: 8 columns (16 fp16)
          mma_ts(tmem + kOCol, pc + 8u * j, dh + (uint32_t)(j * (2048 >> 4)), hi32, idesc(D, true), j ? 1u : (uint32_t)i);
        commit(bar0 + 8 * (kBarVEmpty + (i & 1)));
        commit(bar0 + 8 * (kBarO + (i & 3)));
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax: thread = query row ----------------
    const int group = warp >> 2, part = warp & 3, r = part * 32 + lane, row = row0 + r;
    const bool row_ok = row < a.rows;
    const bool live = row0 + part * 32 < a.rows;
    const uint32_t lanes = (uint32_t)(part * 32) << 16;
    const int t = row_ok ? row / a.gqa : 0, h = hk * a.gqa + (row_ok ? row % a.gqa : 0);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    query_rows();
    bool ok = wait_warp(bar0 + 8 * kBarQ, 0);
    if (!ok) atomicCAS(err, 0, 62 | (10 << 8));
    // scores stay in the products' unit (additive masks: natural units) up to their difference to the reference, so that scores of
    // any size tell their order; the unit is never 0 (a scale of 0): a hidden score stays -inf under it
    auto unit_of_scores = [&]() {
      const int eq = sE[r];
      return fminf(fmaxf(fabsf(a.scale) * pow2(eq >= kOdd / 2 ? eq - kOdd : eq) * pow2(kUnit), 1e-37f), 2e38f);
    };
    const bool odd = kMask >= 2 && __any_sync(0xffffffffu, sE[r] >= kOdd / 2);
    const float c = kMask >= 2 ? unit_of_scores() : 1.f, cl = (kMask >= 2 ? 1.f : unit_of_scores()) * kLog2e;
    // last key the row sees; rows behind the last one compute what nobody reads
    const int lim = row_ok ? min(len - a.T + t, hi - 1) : live ? hi - 1 : -1;
    long long mat = row_ok ? b * a.m_sb + h * a.m_sh + t * a.m_st : 0;   // its mask row, or that of the warp's first row
    const long long mat0 = __shfl_sync(0xffffffffu, mat, 0);
    if (!row_ok) mat = mat0;
    const bool shared = kMask == 1 && __all_sync(0xffffffffu, mat == mat0);
    float m_l = -INFINITY, l = 0.f;   // this half's sum and the reference it is relative to
    // A tile; false where nothing may follow it.  The usual form gives up, with nothing changed, at the first tile that holds unusual keys
    // or values or whose rows carry exponents; from there on the general form takes the range, tile after tile.  What those need goes
    // through tensor memory in rolled loops.  (In one form with branches the usual tiles took 3 to 5 % longer.)
    bool placed = false;   // the tile's scores have their mask already
    auto tile = [&](int i, auto general) -> bool {
      constexpr bool kGeneral = decltype(general)::value;
      const int n0 = order.base(i >> 1) + ((i & 1) * kTile ^ order.flip(i >> 1));
      uint32_t bits[2];                  // the mask, on its way before the scores are waited for (fp32: below)
      uint32_t words[(kMask == 3 ? 16 : kTile / 2) + 4];
      if constexpr (kMask == 1) mask_bits(a, mat, shared, n0, lim, hi, bits);
      if constexpr (kMask == 2) mask_entries<T, kTile / 2>(a, mat, n0, lim, words);
      if constexpr (kMask == 3) mask_entries<float, 16>(a, mat, n0, lim, words);
      if (!wait_warp(bar0 + 8 * (kBarS + ((i >> 1) & 1)), (i >> 2) & 1)) { atomicCAS(err, 0, 62 | (6 << 8)); ok = false; return false; }
      fence_after();
      if (!live) {   // P is whatever is there: lanes of their own
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar0 + 8 * (kBarP + (i & 3)));
        return true;
      }
      const uint32_t s_col = tmem + lanes + 64u * (i & 3);
      const Meta& mt = meta[(i >> 1) & (kMeta - 1)];
      const int blk = 2 * (i & 1);   // the tile's 32-key blocks in `mt`: blk and blk + 1
      const bool k_odd = *(const uint64_t*)(mt.k_odd + blk) != 0;
      if (!kGeneral && k_odd) return false;
      if (kGeneral && k_odd) {
#pragma unroll 1
        for (int e0 = 0; e0 < kTile; e0 += 16) {
          uint32_t x[16];
          ld16(s_col + e0, x);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * own_power(mt, 32 * blk + e0 + e));
          st16(s_col + e0, x);
        }
        wait_st();
      }
      if (kMask >= 2 && !(kGeneral && placed)) {   // scaled score + mask back into place, 16 at a time: with the entries, all 64 would not fit the registers
        const bool careful = odd || k_odd || __any_sync(0xffffffffu, c > 1e28f);
        uint32_t x[2][16];
        ld16(s_col, x[0]);
#pragma unroll
        for (int e0 = 0; e0 < kTile; e0 += 16) {
          uint32_t(&y)[16] = x[(e0 >> 4) & 1];
          if constexpr (kMask == 3) if (e0) mask_entries<float, 16>(a, mat, n0 + e0, lim, words);
          wait_ld();
          if (e0 + 16 < kTile) ld16(s_col + e0 + 16, x[((e0 >> 4) & 1) ^ 1]);
          auto entry = [&](int e) {
            return kMask == 3 ? __uint_as_float(words[e]) : TR::bits_to_float((uint16_t)(words[((e0 + e) >> 1) & 31] >> (16 * (e & 1))));
          };
          if (careful) {   // a hidden key stays hidden under a score that is not finite
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (entry(e) == -INFINITY) y[e] = 0;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(fmaf(__uint_as_float(y[e]), c, entry(e)));
          st16(s_col + e0, y);
        }
        wait_st();
      }
      uint32_t v[kTile];
      ld32(s_col, v);
      ld32(s_col + 32, v + 32);
      // every key of the tile seen by every row of the warp (additive masks aside)
      const bool plain = __all_sync(0xffffffffu, n0 + kTile - 1 <= lim && (kMask != 1 || (bits[0] & bits[1]) == 0xFFFFFFFFu));
      if (!wait_warp(bar0 + 8 * (kBarVMeta + ((i >> 1) & (kMeta - 1))), (i / (2 * kMeta)) & 1)) { atomicCAS(err, 0, 62 | (13 << 8)); ok = false; }
      wait_ld();
      if (!ok) return false;
      if (!plain) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t seen = seen_bits(n0 + 32 * q, lim);
          if (kMask == 1) seen &= bits[q];
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((seen >> e) & 1)) v[32 * q + e] = 0xFF800000u;
        }
      }
      bool own = *(const uint64_t*)(mt.v_odd + blk) != 0;   // the rows' exponents come into play
      if (!kGeneral && own) {
        placed = kMask >= 2;
        return false;
      }
      float top = -INFINITY;
      {
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int e = 0; e < kTile; e += 4) {
          t0 = fmaxf(fmaxf(t0, __uint_as_float(v[e])), __uint_as_float(v[e + 1]));
          t1 = fmaxf(fmaxf(t1, __uint_as_float(v[e + 2])), __uint_as_float(v[e + 3]));
        }
        top = fmaxf(t0, t1);
      }
      // ---- the row's reference: what the tile before left, moved when this tile exceeds it by 8 octaves ----
      float m = -INFINITY, ev = 0.f;
      if (i > 0) {
        if (!wait_warp(bar0 + 8 * (kBarM + 4 * (group ^ 1) + part), ((i - 1) >> 1) & 1)) { atomicCAS(err, 0, 62 | (12 << 8)); ok = false; return false; }
        m = sRef[r];
        if (sOwn[part] != 0) {
          if (!kGeneral) {
            placed = kMask >= 2;
            return false;
          }
          own = true;
          ev = (float)sEv[r];
        }
      }
      bool grow = (top - m) * cl > 8.f;
      const float now = grow ? top : m;
      float ev_now = ev;
      if (kGeneral && own) {
#pragma unroll
        for (int e0 = 0; e0 < kTile; e0 += 16) st16(s_col + e0, v + e0);
        wait_st();
        float d = -INFINITY;   // octaves of the row's largest p 2^x; NaN counts as none
        bool moves = ev != 0.f;   // a row that sees none of the unusual values, and saw none, stays as it is
        const bool all_move = __all_sync(0xffffffffu, moves);
#pragma unroll 1
        for (int e0 = 0; e0 < kTile; e0 += 16) {
          uint32_t x[16];
          ld16(s_col + e0, x);
          const uint4 xs = own_exponents(mt, 32 * blk + e0);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) d = fmaxf(d, fmaf(__uint_as_float(x[e]) - now, cl, exponent(xs, e)));
          const uint32_t odd16 = mt.v_odd[blk + (e0 >> 5)] >> (e0 & 31) & 0xFFFFu;
          if (!all_move && odd16 != 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) moves = moves || (((odd16 >> e) & 1) && x[e] != 0xFF800000u);
          }
        }
        grow = grow || (moves && d > ev + 9.f);
        if (grow && moves) ev_now = fminf(fmaxf(fmaxf(ceilf(d), ev + floorf((m - now) * cl)), -126.f), 126.f);
      }
      if (__any_sync(0xffffffffu, grow)) {
        const float fo = grow ? ex2(fmaf(m - now, cl, ev - ev_now)) : 1.f;   // a row that does not grow keeps every bit
        if (i > 0) {
          if (!wait_warp(bar0 + 8 * (kBarO + ((i - 1) & 3)), ((i - 1) >> 2) & 1)) { atomicCAS(err, 0, 62 | (7 << 8)); ok = false; return false; }
          fence_after();
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 16) {
            uint32_t o[16];
            ld16(tmem + lanes + kOCol + c0, o);
            wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fo);
            st16(tmem + lanes + kOCol + c0, o);
          }
          wait_st();
        }
      }
      m = now;
      sRef[r] = m;
      if (kGeneral && own) sEv[r] = (int8_t)ev_now;
      if ((kGeneral && own) || i == 0) {
        const bool any = kGeneral && __any_sync(0xffffffffu, ev_now != 0.f);
        if (lane == 0) sOwn[part] = any;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar0 + 8 * (kBarM + 4 * group + part));
      if (m != m_l) {
        if (m_l != -INFINITY) l *= ex2((m_l - m) * cl);
        m_l = m;
      }
      // ---- P ----
      const float ref = m == -INFINITY ? 0.f : m;
      const uint64_t cl2 = pair(cl, cl), ref2 = pair(-ref, -ref), shift2 = pair(kPShift, kPShift);
      uint64_t sum = 0;
      if (kGeneral && own) {
        const float off = kPShift - ev_now;
#pragma unroll 1
        for (int e0 = 0; e0 < kTile; e0 += 16) {
          uint32_t x[16], w[8];
          ld16(s_col + e0, x);
          const uint4 xs = own_exponents(mt, 32 * blk + e0);
          wait_ld();
          const uint32_t bad = mt.v_bad[blk + (e0 >> 5)] >> (e0 & 31);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            // a value that is not finite makes the rows NaN that see its key
            const float x0 = ((bad >> e) & 1) && x[e] != 0xFF800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(x[e]);
            const float x1 = ((bad >> e) & 2) && x[e + 1] != 0xFF800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(x[e + 1]);
            const uint64_t d2 = add2(pair(x0, x1), ref2);
            float p0, p1;
            unpair(fma2(d2, cl2, shift2), p0, p1);
            sum = add2(sum, pair(ex2(p0), ex2(p1)));
            unpair(fma2(d2, cl2, pair(off + exponent(xs, e), off + exponent(xs, e + 1))), p0, p1);
            const __half2 p = __floats2half2_rn(ex2(p0), ex2(p1));
            w[e >> 1] = *(const uint32_t*)&p;
          }
          st8(s_col + (e0 >> 1), w);   // over columns that have been read
        }
      } else {
#pragma unroll
        for (int e0 = 0; e0 < kTile; e0 += 16) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const uint64_t d2 = add2(pair(__uint_as_float(v[e0 + e]), __uint_as_float(v[e0 + e + 1])), ref2);
            float p0, p1;
            unpair(fma2(d2, cl2, shift2), p0, p1);
            p0 = ex2(p0);
            p1 = ex2(p1);
            sum = add2(sum, pair(p0, p1));
            const __half2 p = __floats2half2_rn(p0, p1);
            w[e >> 1] = *(const uint32_t*)&p;
          }
          st8(s_col + (e0 >> 1), w);   // over columns that are in registers
        }
      }
      {
        float sum0, sum1;
        unpair(sum, sum0, sum1);
        l = fmaf(sum0 + sum1, 1.f / 64.f, l);
      }
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar0 + 8 * (kBarP + (i & 3)));
      placed = false;
      return true;
    };
    int i = group;
    while (i < tiles && ok && tile(i, std::false_type{})) i += 2;
    while (i < tiles && ok && tile(i, std::true_type{})) i += 2;
    // ---- epilogue: either half of the softmax takes half of the channels; a warp's 32 rows go through shared memory (all of Q, K
    // and V is spent), so that they leave as whole lines ----
    // The last product.  First the last scores: with an odd number of tiles the second half has none of that pair and may be early, while
    // the product four before the last one is still out and the phase could be mistaken; the scores took that one's columns.  Behind both
    // waits every code has been unpacked, so their buffer is free for sEnd.
    if (tiles > 0 && ok && !(wait_warp(bar0 + 8 * (kBarS + ((pairs - 1) & 1)), ((pairs - 1) >> 1) & 1) &&
                             wait_warp(bar0 + 8 * (kBarO + ((tiles - 1) & 3)), ((tiles - 1) >> 2) & 1))) { atomicCAS(err, 0, 62 | (8 << 8)); ok = false; }
    fence_after();
    sEnd[group * kRows + r] = make_float2(m_l, l);
    named_bar_sync(1, 256);
    const bool have = tiles > 0 && ok;
    if (live) {
      const float m = tiles > 0 ? sRef[r] : -INFINITY;
      const int ev = tiles > 0 && sOwn[part] != 0 ? sEv[r] : 0;
      l = 0.f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float2 x = sEnd[g * kRows + r];
        l = fmaf(x.y, x.x == -INFINITY ? 1.f : ex2((x.x - m) * cl), l);
      }
      const bool last = a.splits == 1;
      const float inv = l == 0.f ? 1.f : 1.f / l, nan = l * 0.f;   // a row that sees nothing yields zeros; NaN reaches the whole row
      // over the range's own sum before the exponent comes back: a sum of large values may be no fp32 number
      const float over = pow2(kUnit - (int)kPShift) * inv, undo = pow2(ev);
      const size_t at = ((size_t)bhk * a.rows + row) * a.splits + split;
      uint8_t* stage = smem + r * (D * 4 + 16);   // rows 16 bytes apart modulo 128: no bank conflicts
      const int c_first = group * (D / 2);
#pragma unroll 1
      for (int c0 = c_first; c0 < c_first + D / 2; c0 += 32) {
        uint32_t o[32];
        if (have) {
          ld32(tmem + lanes + kOCol + c0, o);
          wait_ld();
        }
        float y[32];   // back to the channels' order
#pragma unroll
        for (int e = 0; e < 32; ++e) y[(e & ~7) + ((e & 1) << 2) + ((e & 7) >> 1)] = have ? __uint_as_float(o[e]) * over * undo : 0.f;
        if (last) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            T z[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) z[x] = TR::from_float(nan == 0.f ? y[e + x] : nan);
            *(uint4*)(stage + (c0 + e) * 2) = *(const uint4*)z;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *(float4*)(stage + (c0 + e) * 4) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
        }
      }
      if (row_ok && !last && group == 0) {
        a.part_m[at] = kMask >= 2 ? m : m * unit_of_scores();
        a.part_l[at] = l;
      }
      const int bytes = D / 2 * (last ? 2 : 4);   // of half a row: 512, 256 or 128
      const uint64_t dst = (uint64_t)(last ? (const uint8_t*)((T*)a.out + out_row(a, b, hk, row) * D) : (const uint8_t*)(a.part_o + at * D)) +
                           group * bytes;
      const int per = 512 / bytes;                // rows a warp stores at once
      const int off = lane * 16 & (bytes - 1);
      __syncwarp();
#pragma unroll 8
      for (int r1 = 0; r1 < 32; r1 += per) {
        const int rr = r1 + lane * 16 / bytes;
        const uint64_t to = __shfl_sync(0xffffffffu, dst, rr);
        const uint4 x = *(const uint4*)(smem + (part * 32 + rr) * (D * 4 + 16) + group * bytes + off);
        if (row0 + part * 32 + rr < a.rows) *(uint4*)(to + off) = x;
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kIssuer)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

template <typename T, int D>
int launch(const SdpaArgs& a, cudaStream_t st, int device) {
  constexpr size_t tiles = (size_t)3 * (D / kGroup) * kSlab, rest = (size_t)kKeys * D + kBars * 8 + kMeta * sizeof(Meta) + kRows * 7 + 32;
  static_assert(kRows * (D * 4 + 16) <= tiles, "the epilogue's rows fit where Q, K and V were");
  constexpr size_t smem = tiles + rest;
  static_assert(smem <= 227 * 1024, "shared memory");
  const int mask = a.mask_kind;   // 0 .. 3
  auto kern = mask == 0 ? kv4_sdpa_tc_kernel<T, D, 0> : mask == 1 ? kv4_sdpa_tc_kernel<T, D, 1> :
              mask == 2 ? kv4_sdpa_tc_kernel<T, D, 2> : kv4_sdpa_tc_kernel<T, D, 3>;
  static std::mutex mu;
  static bool done[64][4] = {};
  {
    std::lock_guard<std::mutex> lk(mu);
    bool& d = done[device & 63][mask];
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
