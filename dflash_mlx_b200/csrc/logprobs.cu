// Log-probabilities of given tokens, entropy and the top alternatives of every row of logits, in one pass over the logits.
//
//   m = max x,  y = (x - m) log2(e) / T,  L = sum 2^y,  W = sum y 2^y
//   log p[token] = (x[token] - m) / T - ln L,   entropy = ln L - ln 2 W / L
// Every thread sums relative to the maximum of its own elements, with one fma for y (the rounding of m log2(e) / T is taken back
// from the sums afterwards), and the (m, L, W) triples are merged in a fixed tree (L' = L 2^d, W' = (W + d L) 2^d with d = (m - m')
// log2(e) / T), so the result does not depend on timing.
//
// A block passes over its share of the row, 32 (16-bit types) or 16 elements a thread at a time, the next ones on their way.
// Top alternatives: 64 groups of threads (of those that a short row fills) give 64 maxima; at least top_k elements are >= the top_k-th largest of them, and only
// those (a few dozen of tens of thousands) are collected and ranked by counting.  Keys are (value, lower index first) and
// therefore unique.  The first pass sets the bar that way, later passes collect what beats the k-th best so far; the list is ranked
// after passes 1, 4, 16 ... and the last, between which nothing waits.  If it overflows there, the row starts over with a
// ranking after every pass; when one pass alone collects more than the list holds (a row of equal values, sorted logits) the top_k-th largest key is
// found bit by bit.
//
// One row per thread-block cluster: one block a row when rows alone fill the SMs, up to eight otherwise, whose triples and lists the
// first block merges through distributed shared memory.  Measured (bf16, 151936 logits): 1999 rows with suppressed tokens and 5
// alternatives 213 us (2.9 TB/s, HBM floor 93: issue slots 69 % busy, exponentials 38 % of their pipe, the rest waits at the rankings'
// barriers), 16 rows with 20 alternatives 16.5 us (latency: passes, ranking, cluster merge).
#include <cooperative_groups.h>

#include <mutex>

#include "common.cuh"

namespace dflash {
namespace lp {
namespace {

constexpr int kThreads = 256, kGroups = 64, kMaxK = 32, kList = 1024, kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* logits;
  long long ld;
  const int* tokens;
  const uint8_t* suppress;
  float* token_logprob;
  float* entropy;
  float* top_logprobs;
  int* top_ids;
  double inv_t;                // 1 / temperature
  float scale;                 // log2(e) / temperature
  int V, k;
};

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int kPer = 4, kSlots = 4;
  static constexpr uint32_t kNegInf = 0xFF800000u;
  __device__ static __forceinline__ float get(const uint32_t (&w)[4], int e) { return __uint_as_float(w[e]); }
  __device__ static __forceinline__ void hide(uint32_t (&w)[4], int e) { w[e] = kNegInf; }
  __device__ static __forceinline__ uint2 suppress_bytes(const uint8_t* p) { return make_uint2(*(const uint32_t*)p, 0); }
  __device__ static __forceinline__ void hide_by(uint32_t (&w)[4], uint2 u) {   // the elements whose byte is not 0
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((u.x >> (8 * e)) & 0xFFu) w[e] = kNegInf;
  }
  // whether clamped() keeps a thread's sums right: the clamp is 0 probability next to the maximum m
  __device__ static __forceinline__ bool can_clamp(float, float) { return false; }
  __device__ static __forceinline__ uint32_t clamped(uint32_t w) { return w; }
  __device__ static __forceinline__ void two(uint32_t, float&, float&) {}
  __device__ static __forceinline__ void put(uint32_t (&w)[4], int e, const float* p) { w[e] = __float_as_uint(*p); }
  __device__ static __forceinline__ float load(const float* p) { return *p; }
  __device__ static __forceinline__ float max_of(const uint32_t (&w)[kSlots][4]) {   // NaN is passed over
    float m = -INFINITY;
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = fmaxf(m, __uint_as_float(w[s][i]));
    return m;
  }
};
__device__ __forceinline__ __nv_bfloat162 as_pair(uint32_t u, __nv_bfloat16) { return *(const __nv_bfloat162*)&u; }
__device__ __forceinline__ __half2 as_pair(uint32_t u, __half) { return *(const __half2*)&u; }
template <typename T, uint32_t kInf> struct Elem16 {
  static constexpr int kPer = 8, kSlots = 4;
  __device__ static __forceinline__ float get(const uint32_t (&w)[4], int e) {
    return MmaTraits<T>::bits_to_float((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
  }
  __device__ static __forceinline__ void put_bits(uint32_t (&w)[4], int e, uint32_t bits) {
    w[e >> 1] = (e & 1) ? ((w[e >> 1] & 0xFFFFu) | (bits << 16)) : ((w[e >> 1] & 0xFFFF0000u) | bits);
  }
  __device__ static __forceinline__ void hide(uint32_t (&w)[4], int e) { put_bits(w, e, kInf); }
  __device__ static __forceinline__ uint2 suppress_bytes(const uint8_t* p) { return *(const uint2*)p; }
  __device__ static __forceinline__ void hide_by(uint32_t (&w)[4], uint2 u) {
    const uint32_t t[2] = {u.x * 255u, u.y * 255u};   // 0 or 1 -> 0 or 255, byte by byte
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = prmt(t[i >> 1], 0, (i & 1) ? 0x3322 : 0x1100);   // a byte for each half
      w[i] = (w[i] & ~m) | ((kInf | (kInf << 16)) & m);
    }
  }
  // whether clamped() keeps a thread's sums right: the clamp (-1e30, fp16: -65504) has probability 0 next to the maximum m, and the
  // rounding of m * scale, which every y of the thread carries until the end, is no more than 2^-5 octaves
  __device__ static __forceinline__ bool can_clamp(float m, float scale) {
    return scale >= 0.01f && scale < 1e6f && m > -40000.f && fabsf(m * scale) < 1048576.f;
  }
  __device__ static __forceinline__ uint32_t clamped(uint32_t w) {
    const uint32_t low = kInf == 0xFF80u ? 0xF149F149u : 0xFBFFFBFFu;
    const auto m = __hmax2_nan(as_pair(w, T()), as_pair(low, T()));
    return *(const uint32_t*)&m;
  }
  __device__ static __forceinline__ void two(uint32_t w, float& x0, float& x1) {
    x0 = MmaTraits<T>::bits_to_float((uint16_t)w);
    x1 = MmaTraits<T>::bits_to_float((uint16_t)(w >> 16));
  }
  __device__ static __forceinline__ void put(uint32_t (&w)[4], int e, const T* p) { put_bits(w, e, *(const uint16_t*)p); }
  __device__ static __forceinline__ float load(const T* p) { return MmaTraits<T>::to_float(*p); }
  __device__ static __forceinline__ float max_of(const uint32_t (&w)[kSlots][4]) {   // packed; NaN is passed over
    auto m = as_pair(w[0][0], T());
#pragma unroll
    for (int i = 1; i < 4 * kSlots; ++i) m = __hmax2(m, as_pair(w[i >> 2][i & 3], T()));
    return fmaxf(fmaxf(MmaTraits<T>::to_float(m.x), MmaTraits<T>::to_float(m.y)), -INFINITY);
  }
};
template <> struct Elem<__nv_bfloat16> : Elem16<__nv_bfloat16, 0xFF80u> {};
template <> struct Elem<__half> : Elem16<__half, 0xFC00u> {};

struct Sums { float m, l, w; };
__device__ __forceinline__ Sums merge(const Sums& a, const Sums& b, float scale) {
  Sums s;
  s.m = fmaxf(a.m, b.m);
  // a side without a maximum has sums of zero (or NaN, which stays): it needs no factor
  const float da = a.m == -INFINITY ? 0.f : (a.m - s.m) * scale, db = b.m == -INFINITY ? 0.f : (b.m - s.m) * scale;
  const float fa = exp2f(da), fb = exp2f(db);
  s.l = a.l * fa + b.l * fb;
  // a vanished side must not turn an infinite distance into NaN
  s.w = (fa == 0.f ? 0.f : fmaf(da, a.l, a.w) * fa) + (fb == 0.f ? 0.f : fmaf(db, b.l, b.w) * fb);
  return s;
}
// With the lane whose number differs in bit o: the lower lane's triple first, so that both compute the same bits.
__device__ __forceinline__ Sums merge_lanes(const Sums& s, int o, float scale) {
  const Sums other = {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.l, o), __shfl_xor_sync(0xffffffffu, s.w, o)};
  return (threadIdx.x & o) ? merge(other, s, scale) : merge(s, other, scale);
}
__device__ __forceinline__ unsigned long long key_of(float v, int index) {
  const uint32_t u = __float_as_uint(__fadd_rn(v, 0.f));   // -0 and +0 are one value
  const uint32_t o = u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  return ((unsigned long long)o << 32) | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)~(uint32_t)k; }

struct Shared {
  Sums warp_sums[kThreads / 32];
  Sums block_sums;
  float group_max[kGroups];
  float tau;                                      // only elements from here on (the first pass) or beyond (later ones) matter
  int count;
  unsigned long long list[kList];
  unsigned long long top[kMaxK];                  // this block's best, highest first; 0 = none
  unsigned long long gathered[kMaxCluster * kMaxK];         // first block of a cluster: every block's `top`
  int counts[2][kThreads / 32];
  float given;                                    // the given token's logit; NaN outside the vocabulary
  uint4 stage[4][kThreads];                       // elements of threads that hold candidates, to be picked by number
};

// The `k` largest of list[0..n) in order; keys are unique, 0 marks an empty place and is skipped.
__device__ __forceinline__ void rank_into(unsigned long long* top, const unsigned long long* list, int n, int k) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long mine = list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += list[j] > mine;
    if (rank < k && mine != 0) top[rank] = mine;
  }
}

// raw[s] for an s that is not known at compile time (registers cannot be indexed).
template <int N>
__device__ __forceinline__ void slot(const uint32_t (&raw)[N][4], int s, uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i == s) { w[0] = raw[i][0]; w[1] = raw[i][1]; w[2] = raw[i][2]; w[3] = raw[i][3]; }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) token_logprobs_kernel(const Args a) {
  namespace cg = cooperative_groups;
  using E = Elem<T>;
  constexpr int kPer = E::kPer, kSlots = E::kSlots;
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / blocks;
  pdl_wait();
  pdl_trigger();
  const T* x = (const T*)a.logits + row * a.ld;
  // 16-byte vectors from the aligned address at or before the row; the first and last are loaded element by element
  const int skew = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int vecs = (skew + a.V + kPer - 1) / kPer;
  const int share = (vecs + blocks - 1) / blocks;
  const int v0 = me * share, v1 = min(vecs, v0 + share);
  Sums sums = {-INFINITY, 0.f, 0.f}, run = sums;   // run: of the passes that can_clamp, relative to run.m, which `at` stands for
  float at = 0.f;
  if (tid < kMaxK) sh.top[tid] = 0;
  if (tid == 0) sh.count = 0;
  const bool packed = a.suppress != nullptr && skew == 0 && ((uintptr_t)a.suppress & (kPer - 1)) == 0;
  uint2 bytes[kSlots];   // of `suppress`, for the vectors on their way
  auto load = [&](int base, uint32_t (&raw)[kSlots][4]) {
    const int last = base + kThreads * kSlots;
    if (base * kPer >= skew && last <= v1 && last * kPer - skew <= a.V) {   // the whole pass lies inside the row
      const T* px = x + (base + tid) * kPer - skew;
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        const uint4 u = __ldcs((const uint4*)(px + s * kThreads * kPer));
        raw[s][0] = u.x; raw[s][1] = u.y; raw[s][2] = u.z; raw[s][3] = u.w;
        bytes[s] = packed ? E::suppress_bytes(a.suppress + (base + s * kThreads + tid) * kPer) : make_uint2(0, 0);
      }
      return;
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int v = base + s * kThreads + tid;
      const int i0 = v * kPer - skew;
      bytes[s] = make_uint2(0, 0);
      if (packed && v < v1 && i0 + kPer <= a.V) bytes[s] = E::suppress_bytes(a.suppress + i0);
      if (v < v1 && i0 >= 0 && i0 + kPer <= a.V) {
        const uint4 u = __ldcs((const uint4*)(x + i0));
        raw[s][0] = u.x; raw[s][1] = u.y; raw[s][2] = u.z; raw[s][3] = u.w;
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (v < v1 && i0 + e >= 0 && i0 + e < a.V) E::put(raw[s], e, x + i0 + e);
          else E::hide(raw[s], e);
        }
      }
    }
  };
  bool careful = false;
  uint32_t next[kSlots][4];
  if (v0 < v1) load(v0, next);
  if (me == 0 && tid == kThreads - 1) {   // two dependent reads, under the first vectors'
    const int token = a.tokens[row];
    sh.given = token < 0 || token >= a.V ? __int_as_float(0x7FC00000)
               : a.suppress != nullptr && a.suppress[token] ? -INFINITY : E::load(x + token);
  }
  for (int base = v0; base < v1; base += kThreads * kSlots) {
    uint32_t raw[kSlots][4];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[s][i] = next[s][i];
      if (a.suppress != nullptr) {
        const int v = base + s * kThreads + tid;
        const int i0 = v * kPer - skew;
        if (packed && i0 + kPer <= a.V) {   // the vector's bytes at once
          E::hide_by(raw[s], bytes[s]);
        } else if (v < v1) {
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            if (i0 + e >= 0 && i0 + e < a.V && a.suppress[i0 + e]) E::hide(raw[s], e);
        }
      }
    }
    if (base + kThreads * kSlots < v1) load(base + kThreads * kSlots, next);   // in flight under this pass
    const float top = E::max_of(raw);   // of this pass's elements; NaN is passed over
    bool nan = false;                   // whether an element was NaN or +inf
    if (base + warp * 32 >= v1) {   // the warp has nothing of this pass
    } else if (E::can_clamp(top, a.scale)) {   // hidden elements become a finite value of probability 0, two at a time
      if (top > run.m) {                // the thread's reference moves: y' = x scale - at, at = rounded(reference scale)
        const float to = top * a.scale, d = run.m == -INFINITY ? 0.f : at - to, f = exp2f(d);
        run.w = fmaf(d, run.l, run.w) * f;
        run.l *= f;
        run.m = top;
        at = to;
      }
      float l0 = run.l, l1 = 0.f, w0 = run.w, w1 = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * kSlots; ++i) {
        float x0, x1;
        E::two(E::clamped(raw[i >> 2][i & 3]), x0, x1);
        const float y0 = fmaf(x0, a.scale, -at), y1 = fmaf(x1, a.scale, -at);
        const float p0 = exp2f(y0), p1 = exp2f(y1);
        l0 += p0;
        l1 += p1;
        w0 = fmaf(y0, p0, w0);
        w1 = fmaf(y1, p1, w1);
      }
      run.l = l0 + l1;
      run.w = w0 + w1;
      nan = !(run.l == run.l);
    } else {
      Sums mine = {top, 0.f, 0.f};
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const float y = (E::get(raw[s], e) - ref) * a.scale;
          const float p = exp2f(y);
          mine.l += p;
          mine.w = fmaf(fmaxf(y, -1e30f), p, mine.w);   // a hidden element adds 0, not -inf * 0; NaN stays through p
        }
      nan = !(mine.l == mine.l);
      sums = merge(sums, mine, a.scale);
    }
    if (a.k > 0) {
      // ---- candidates of this pass ----
      const bool first = base == v0;
      if (first) {   // everything >= the k-th largest group maximum
        const int wide = v1 - v0 > 2 * kGroups ? 2 : v1 - v0 > kGroups ? 1 : 0;   // 2^wide threads a group: short rows fill few threads
        float g = top;
        for (int o = 1; o < 1 << wide; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if ((lane & ((1 << wide) - 1)) == 0 && tid >> wide < kGroups) sh.group_max[tid >> wide] = g;
        __syncthreads();
        const float g0 = sh.group_max[lane], g1 = sh.group_max[lane + 32];
#pragma unroll
        for (int i = 0; i < kGroups / (kThreads / 32); ++i) {   // every warp ranks its own groups, ties by number
          const int j = warp * (kGroups / (kThreads / 32)) + i;
          const float v = sh.group_max[j];
          const int rank = __popc(__ballot_sync(0xffffffffu, g0 > v || (g0 == v && lane < j))) +
                           __popc(__ballot_sync(0xffffffffu, g1 > v || (g1 == v && lane + 32 < j)));
          if (rank == a.k - 1 && lane == 0) sh.tau = v;
        }
        __syncthreads();
      }
      const float tau = sh.tau;
      // NaN elements count as the largest; a thread whose own maximum does not reach tau can only hold NaN beyond it
      const bool has = ((first ? top >= tau : !(top <= tau)) || nan) && base + tid < v1;
      if (has) {
        uint32_t hits = 0;
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          sh.stage[s][tid] = make_uint4(raw[s][0], raw[s][1], raw[s][2], raw[s][3]);
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const float f = E::get(raw[s], e);
            hits |= (uint32_t)(first ? !(f < tau) : !(f <= tau)) << (s * kPer + e);
          }
          if (base + s * kThreads + tid >= v1) hits &= (1u << (s * kPer)) - 1u;   // nothing from here on
        }
        while (hits) {
          const int at_e = __ffs(hits) - 1, s = at_e / kPer, e = at_e % kPer;
          hits &= hits - 1;
          const int v = base + s * kThreads + tid, i = v * kPer - skew + e;
          if (v < v1 && i >= 0 && i < a.V) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kList - kMaxK) sh.list[at] = key_of(E::load((const T*)&sh.stage[s][tid] + e), i);
          }
        }
      }
      const int pass = (base - v0) / (kThreads * kSlots) + 1;
      if (!careful && ((pass & (pass - 1)) != 0 || (pass & 0x2AAAAAAA) != 0) && base + kThreads * kSlots < v1) continue;
      __syncthreads();
      const int n = sh.count;
      if (n > kList - kMaxK && !careful && !first) {   // over several passes: once more, ranking after each
        __syncthreads();
        careful = true;
        if (tid < kMaxK) sh.top[tid] = 0;
        if (tid == 0) sh.count = 0;
        sums = run = {-INFINITY, 0.f, 0.f};
        at = 0.f;
        base = v0 - kThreads * kSlots;
        load(v0, next);
        continue;
      }
      if (n <= 64) {   // one warp ranks them
        if (warp == 0) {
          const int all = n + (first ? 0 : a.k);   // the best of the earlier passes compete again
          if (!first && lane < a.k) sh.list[n + lane] = sh.top[lane];
          __syncwarp();
          const unsigned long long none = 0, k0 = lane < all ? sh.list[lane] : none, k1 = lane + 32 < all ? sh.list[lane + 32] : none,
                                   k2 = lane + 64 < all ? sh.list[lane + 64] : none;
          sh.top[lane] = 0;
          int r0 = 0, r1 = 0, r2 = 0;
#pragma unroll 4
          for (int j = 0; j < all; ++j) {
            const unsigned long long q = sh.list[j];
            r0 += q > k0;
            r1 += q > k1;
            r2 += q > k2;
          }
          __syncwarp();
          if (k0 != 0 && r0 < a.k) sh.top[r0] = k0;
          if (k1 != 0 && r1 < a.k) sh.top[r1] = k1;
          if (k2 != 0 && r2 < a.k) sh.top[r2] = k2;
        }
      } else if (n <= kList - kMaxK) {
        int all = n;
        if (!first) {
          if (tid < a.k) {
            sh.list[n + tid] = sh.top[tid];
            sh.top[tid] = 0;
          }
          all += a.k;
          __syncthreads();
        }
        rank_into(sh.top, sh.list, all, a.k);
      } else {
        // too many at or above tau (ties, sorted logits): the k-th largest key bit by bit, then exactly the keys from it on
        const unsigned long long earlier = tid < kMaxK ? sh.top[tid] : 0ull;
        unsigned long long kth = 0;
#pragma unroll 1
        for (int bit = 63; bit >= 0; --bit) {
          const unsigned long long t = kth | (1ull << bit);
          int n_at = earlier >= t;
#pragma unroll 1
          for (int s = 0; s < kSlots; ++s) {
            uint32_t w[4];
            slot(raw, s, w);
            const int v = base + s * kThreads + tid, i0 = v * kPer - skew;
#pragma unroll
            for (int e = 0; e < kPer; ++e)
              n_at += v < v1 && i0 + e >= 0 && i0 + e < a.V && key_of(E::get(w, e), i0 + e) >= t;
          }
          n_at = __reduce_add_sync(0xffffffffu, n_at);
          if (lane == 0) sh.counts[bit & 1][warp] = n_at;
          __syncthreads();
          n_at = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? sh.counts[bit & 1][lane] : 0);
          if (n_at >= a.k) kth = t;
        }
        if (tid == 0) sh.count = 0;
        if (tid < kMaxK) sh.top[tid] = 0;
        __syncthreads();
        // kth = 0: fewer than k elements so far, all of them stay
        if (earlier >= kth && earlier != 0) sh.list[atomicAdd(&sh.count, 1)] = earlier;
#pragma unroll 1
        for (int s = 0; s < kSlots; ++s) {
          uint32_t w[4];
          slot(raw, s, w);
          const int v = base + s * kThreads + tid, i0 = v * kPer - skew;
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            if (v < v1 && i0 + e >= 0 && i0 + e < a.V) {
              const unsigned long long q = key_of(E::get(w, e), i0 + e);
              if (q >= kth) sh.list[atomicAdd(&sh.count, 1)] = q;
            }
        }
        __syncthreads();
        rank_into(sh.top, sh.list, sh.count, a.k);
      }
      __syncthreads();   // every warp has read the count
      // the next pass: only what beats the k-th best (its own index is lower); -inf while there are fewer than k
      if (tid == 0) {
        sh.count = 0;
        sh.tau = sh.top[a.k - 1] == 0 ? -INFINITY : key_value(sh.top[a.k - 1]);
      }
      __syncthreads();
    }
  }
  if (run.m != -INFINITY) {   // y' was taken from the rounded product: back to the exact one
    const float off = fmaf(run.m, a.scale, -at), z = off * 0.6931471805599453f;
    const float f = fabsf(z) < 0.01f ? fmaf(z, fmaf(z, 0.5f, -1.f), 1.f) : exp2f(-off);
    run.w = fmaf(-off, run.l, run.w) * f;
    run.l *= f;
    sums = merge(sums, run, a.scale);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sums = merge_lanes(sums, o, a.scale);
  if (lane == 0) sh.warp_sums[warp] = sums;
  __syncthreads();
  if (warp == 0) {
    sums = sh.warp_sums[lane & (kThreads / 32 - 1)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1) sums = merge_lanes(sums, o, a.scale);
    if (lane == 0) sh.block_sums = sums;
  }
  if (blocks > 1) cluster.sync();
  else __syncthreads();
  if (me == 0) {
    Sums all = sh.block_sums;
    if (blocks > 1) {   // every lane fetches a block's, all at once
      all = *cluster.map_shared_rank(&sh.block_sums, lane & (blocks - 1));
      for (int o = blocks / 2; o > 0; o >>= 1) all = merge_lanes(all, o, a.scale);
    }
    if (a.k > 0) {
      if (blocks > 1) {
        // a key's rank: its place in its own block's list, and in each other list (sorted, 0 at the end) the number above it
        static_assert(kMaxCluster * kMaxK == kThreads, "a thread per gathered key");
        const int from = warp, place = lane;
        if (from < blocks) sh.gathered[tid] = cluster.map_shared_rank(&sh.top[0], from)[place];
        __syncthreads();
        const unsigned long long mine = from < blocks ? sh.gathered[tid] : 0;
        if (mine != 0) {
          int rank = place;
          for (int o = 0; o < blocks; ++o) {
            if (o == from) continue;
            const unsigned long long* other = sh.gathered + o * kMaxK;
            int above = 0;
#pragma unroll
            for (int step = kMaxK / 2; step > 0; step >>= 1)
              if (other[above + step - 1] > mine) above += step;
            rank += above + (other[above] > mine);
          }
          if (rank < a.k) sh.list[rank] = mine;   // list: free again
        }
        __syncthreads();
      } else {
        if (tid < kMaxK) sh.list[tid] = sh.top[tid];
        __syncthreads();
      }
    }
    const bool empty = all.m == -INFINITY && all.l == 0.f;   // nothing but -inf
    if (tid <= a.k) {
      // tid 0: the given token and the entropy; tid 1..k: an alternative each.  ln L in double: a peaked row has L = 1 + eps
      const double log_l = log((double)all.l);
      const float value = tid == 0 ? sh.given : key_value(sh.list[tid - 1]);
      float out = empty ? -INFINITY : (float)((double)(value - all.m) * a.inv_t - log_l);
      if (tid == 0 && value != value) out = value;
      if (tid == 0) {
        a.token_logprob[row] = out;
        if (a.entropy != nullptr)
          a.entropy[row] = empty ? 0.f : (float)(log_l - (double)(0.69314718056f * (all.w / all.l)));
      } else {
        a.top_logprobs[row * a.k + tid - 1] = out;
        a.top_ids[row * a.k + tid - 1] = key_index(sh.list[tid - 1]);
      }
    }
  }
  if (blocks > 1) cluster.sync();   // the first block has read the others' shared memory
}

template <typename T>
int launch(const Args& a, int R, cudaStream_t st, int device) {
  // rows alone fill the SMs: a block per row passes over it, most passes finding no new candidate; few rows: the cluster grows
  // while a block keeps 2048 elements
  int c = 1;
  while (c < kMaxCluster && (long long)R * c < sm_count(device) && a.V >= 2 * c * 2048) c <<= 1;
  if ((long long)R * c > 0x7fffffffll) return fail(DFLASH_ERR_BAD_SHAPE, "token_logprobs: too many rows");
  cudaError_t e = launch_kernel_cluster(token_logprobs_kernel<T>, dim3((unsigned)R * c), dim3(kThreads), c, 0, st, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? DFLASH_OK : fail(DFLASH_ERR_LAUNCH, "token_logprobs launch: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace lp
}  // namespace dflash

using namespace dflash;

extern "C" int dflash_token_logprobs(const void* logits, long long ld, const int* tokens, const uint8_t* suppress, float temperature,
                                     float* token_logprob, float* entropy, float* top_logprobs, int* top_ids, int R, int V,
                                     int top_k, int dtype, void* stream) {
  if (R < 0 || V < 1 || ld < V) return fail(DFLASH_ERR_BAD_SHAPE, "token_logprobs: R=%d V=%d ld=%lld", R, V, ld);
  if (V > 0x7fffffff - 64 * 1024) return fail(DFLASH_ERR_BAD_SHAPE, "token_logprobs: V=%d too large", V);
  if (top_k < 0 || top_k > lp::kMaxK || top_k > V) return fail(DFLASH_ERR_BAD_SHAPE, "token_logprobs: top_k=%d outside 0..min(%d, V)", top_k, lp::kMaxK);
  // log2(e) / temperature has to be a normal number: the kernels flush others to 0, and -inf * 0 is NaN
  if (!(temperature >= 1e-30f) || !(temperature <= 1e38f)) return fail(DFLASH_ERR_BAD_ARG, "token_logprobs: temperature outside 1e-30..1e38");
  if (R == 0) return DFLASH_OK;
  if (!logits || !tokens || !token_logprob || (top_k > 0 && (!top_logprobs || !top_ids))) return fail(DFLASH_ERR_BAD_ARG, "token_logprobs: null operand");
  const int size = dtype == DFLASH_F32 ? 4 : 2;
  if ((uintptr_t)logits % size) return fail(DFLASH_ERR_MISALIGNED, "token_logprobs: logits are not aligned to their type");
  lp::Args a{logits, ld, tokens, suppress, token_logprob, entropy, top_logprobs, top_ids, 1.0 / (double)temperature, lp::kLog2e / temperature, V, top_k};
  int device = 0;
  cudaGetDevice(&device);
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DFLASH_BF16: return lp::launch<__nv_bfloat16>(a, R, st, device);
    case DFLASH_F16: return lp::launch<__half>(a, R, st, device);
    case DFLASH_F32: return lp::launch<float>(a, R, st, device);
  }
  return fail(DFLASH_ERR_BAD_ARG, "token_logprobs: dtype %d", dtype);
}
