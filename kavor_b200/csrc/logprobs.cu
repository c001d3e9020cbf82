// Log probabilities of given tokens, their ranks, each row's entropy and its
// most likely alternatives, from one pass over the logits.
//
// With m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):
//   logprob_i = (x_i - m) - log S,   entropy = log S - T / S
// (summed against a reference within 10 of the maximum, so at most 10 cancels). An entry of
// -inf has probability 0 and adds 0 to both sums; a row of only -inf has
// logprob -inf and entropy 0. A row with a NaN or +inf has NaN for each.
// Order of the entries: higher logit first, NaN above everything, the lower
// index on ties (-0 equals +0); rank counts the entries before the token.
//
// A cluster of 1..8 CTAs takes a row, each CTA a contiguous part of it in
// 16-byte vectors, four per thread in flight. Every thread keeps its own
// reference r near its maximum (moved only when an entry passes r + 10, so the
// usual vector costs no rescale) and sums S and T against it in 32 bits, with
// packed 2 x fp32 arithmetic. The alternatives come from the same pass: the
// k-th largest of the warps' four largest first maxima is a lower bound of the
// k-th largest entry, so each thread marks those of its vectors that reach it
// (a few hundred of 19 thousand), one bit each, and only they are looked at again
// at the end, when warps sort and merge their entries in 32-entry runs. The rank is counted
// only in steps where a vector's maximum reaches the token's logit.
//
// Measured at 151936 bf16 entries: 2000 rows with 5 alternatives 132 us (4.6 TB/s),
// without 118 us; bound by instructions (8 to 10 an entry, of which one exponential)
// and a row's fixed end (join, expansion and sort: a fifth of a CTA's time), not
// by HBM. 256 rows with 20 alternatives 33 us, 16 rows 12 us: one wave, its fixed ends
// not hidden behind another row's stream.
#include <cuda_fp16.h>

#include "common.cuh"
#include "../../include/kavor_b200.h"

KVB_DEFINE_ERROR_WORD(logprobs)

#include "tcgen05.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kCap = 2048;      // entries of the candidate list
constexpr float kSlack = 10.f;  // how far an entry may pass a thread's reference
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// The largest magnitude a reference r may have. Powers are taken against c = r log2(e)
// rounded to 32 bits; c's residue, half a unit of its last place, is up to 4 at 2^26,
// so the powers lie in 2^+-(4 + 10 log2(e)). (At 1e10 it is 512: 2^y is infinite or 0.)
// Parts whose largest entry is beyond it are summed again entry by entry.
constexpr float kFar = 67108864.f;

// ------------------------------------------------------------ element types
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static constexpr float kFloor = -1e38f;
  static __device__ __forceinline__ uint32_t floor_word(uint32_t w) {
    return __float_as_uint(fmaxf(__uint_as_float(w), kFloor));
  }
  // the largest entry, NaN if there is one
  static __device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
    float a;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(__uint_as_float(x)), "f"(__uint_as_float(y)));
    return __float_as_uint(a);
  }
  static __device__ __forceinline__ float value(uint32_t x) { return __uint_as_float(x); }
  // a bound, and whether an entry reaches it (NaN does)
  static __device__ __forceinline__ uint32_t bound(float x) { return __float_as_uint(x); }
  static __device__ __forceinline__ bool reaches(uint32_t x, uint32_t b) { return !(value(x) < value(b)); }
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  // entries that reach a bound, NaN among them
  static __device__ __forceinline__ unsigned count(const uint4& r, uint32_t b) {
    return (unsigned)reaches(r.x, b) + reaches(r.y, b) + reaches(r.z, b) + reaches(r.w, b);
  }
  // the bound that only entries above b's value reach (not for NaN or +inf)
  static __device__ __forceinline__ uint32_t above(uint32_t b) {
    const uint32_t u = b == 0x80000000u ? 0u : b;
    return u & 0x80000000u ? u - 1 : u + 1;
  }
};

// one bit per 16-bit half of four compare masks
__device__ __forceinline__ unsigned count_masks(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __popc((a & 0x00010001u) | (b & 0x00020002u) | (c & 0x00040004u) | (d & 0x00080008u));
}
template <>
struct Vec<bf16> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static constexpr float kFloor = -9.96920997e37f;
  static __device__ __forceinline__ uint32_t floor_word(uint32_t w) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xfe96fe96u));
    return r;
  }
  // of two entries each, the larger ones in their halves; NaN if there is one
  static __device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
    uint32_t a;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(x), "r"(y));
    return a;
  }
  static __device__ __forceinline__ float value(uint32_t x) {
    float hi = __uint_as_float(x & 0xffff0000u), lo = __uint_as_float(x << 16);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(lo));
    return hi;
  }
  static __device__ __forceinline__ uint32_t bound(float x) {  // never above x
    const uint32_t h = __bfloat16_as_ushort(__float2bfloat16_rd(x));
    return h | h << 16;
  }
  static __device__ __forceinline__ bool reaches(uint32_t x, uint32_t b) {
    uint32_t r;
    asm("{\n\t.reg .pred p, q;\n\tsetp.geu.bf16x2 p|q, %1, %2;\n\tor.pred p, p, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"(x), "r"(b));
    return r != 0;
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float one(const bf16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ unsigned count(const uint4& r, uint32_t b) {
    const __nv_bfloat162 t = *reinterpret_cast<const __nv_bfloat162*>(&b);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    return count_masks(__hgeu2_mask(h[0], t), __hgeu2_mask(h[1], t), __hgeu2_mask(h[2], t), __hgeu2_mask(h[3], t));
  }
  static __device__ __forceinline__ uint32_t above(uint32_t b) {  // both halves alike
    const uint32_t u = (b & 0xffffu) == 0x8000u ? 0u : b & 0xffffu, h = u & 0x8000u ? u - 1 : u + 1;
    return h | h << 16;
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static constexpr float kFloor = -65504.f;
  static __device__ __forceinline__ uint32_t floor_word(uint32_t w) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xfbfffbffu));
    return r;
  }
  // of two entries each, the larger ones in their halves; NaN if there is one
  static __device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
    uint32_t a;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(a) : "r"(x), "r"(y));
    return a;
  }
  static __device__ __forceinline__ float value(uint32_t x) {
    float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(f.x) : "f"(f.y));
    return f.x;
  }
  static __device__ __forceinline__ uint32_t bound(float x) {  // never above x
    const uint32_t h = __half_as_ushort(__float2half_rd(x));
    return h | h << 16;
  }
  static __device__ __forceinline__ bool reaches(uint32_t x, uint32_t b) {
    uint32_t r;
    asm("{\n\t.reg .pred p, q;\n\tsetp.geu.f16x2 p|q, %1, %2;\n\tor.pred p, p, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"(x), "r"(b));
    return r != 0;
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ unsigned count(const uint4& r, uint32_t b) {
    const __half2 t = *reinterpret_cast<const __half2*>(&b);
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    return count_masks(__hgeu2_mask(h[0], t), __hgeu2_mask(h[1], t), __hgeu2_mask(h[2], t), __hgeu2_mask(h[3], t));
  }
  static __device__ __forceinline__ uint32_t above(uint32_t b) {  // both halves alike
    const uint32_t u = (b & 0xffffu) == 0x8000u ? 0u : b & 0xffffu, h = u & 0x8000u ? u - 1 : u + 1;
    return h | h << 16;
  }
};

// A vector's largest entry, as larger() leaves it.
template <typename T>
__device__ __forceinline__ uint32_t largest(const uint4& r) {
  return Vec<T>::larger(Vec<T>::larger(r.x, r.y), Vec<T>::larger(r.z, r.w));
}

// ------------------------------------------------------------------- order
// Whole number whose order is the order of the logits: NaN highest, -0 = +0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0xffffffffu) return NAN;
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// Entries in order: larger is earlier. Distinct for every index, never 0.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  return (uint64_t)order_of(x) << 32 | (uint32_t)(0x7fffffff - i);
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// One step of a bitonic network over the lanes: the pair (lane, lane ^ o)
// keeps its larger key in the lower lane (desc) or in the higher one.
__device__ __forceinline__ uint64_t exchange(uint64_t v, int o, bool desc) {
  const uint64_t w = shfl_xor64(v, o);
  const bool take_max = ((threadIdx.x & o) == 0) == desc;
  return (v > w) == take_max ? v : w;
}
__device__ __forceinline__ uint64_t sort32(uint64_t v) {  // descending over the lanes
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int o = k >> 1; o > 0; o >>= 1) v = exchange(v, o, (lane & k) == 0);
  return v;
}
// The 32 largest of two descending runs, descending.
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b) {
  const uint64_t rb = __shfl_sync(0xffffffffu, b, 31 - (threadIdx.x & 31));
  uint64_t v = a > rb ? a : rb;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = exchange(v, o, true);
  return v;
}

// ------------------------------------------------------------------ shared
struct Stats {
  float m, s, t;  // reference (the largest of the threads'), sums against it; m = -inf: nothing finite
  unsigned rank, bad;
};
struct Shared {
  uint64_t list[kCap];  // candidates
  int vecs[kCap];       // vectors that hold one
  uint64_t run[kWarps][32];
  uint64_t top[32];     // this CTA's largest entries, descending, padded with 0
  Stats warp[kWarps];
  Stats cta;
  unsigned count, noted;
  uint32_t four[32], maxes[kWarps];
};

// The 32 largest keys of the block, each warp holding one descending run;
// the result is in every lane of warp 0 and in sh.top.
__device__ __forceinline__ void block_merge(Shared& sh, uint64_t v, int runs) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int half = runs >> 1; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) sh.run[warp][lane] = v;
    __syncthreads();
    if (warp < half) v = merge32(v, sh.run[warp + half][lane]);
  }
  if (warp == 0) sh.top[lane] = v;
  __syncthreads();
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void un2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// One thread's sums against its reference r, in powers of two: with L =
// log2(e) and c = -r L, S = sum 2^y and T = sum 2^y y over y = x L + c, one FMA
// per entry. c is rounded; its residue is put right in the end. S and T hold two
// partial sums each.
struct Sums {
  float r = 0.f, lim = -INFINITY;  // entries above lim move r; lim = -inf: no entry has made a reference yet
  uint64_t c = 0, S = 0, T = 0;
  bool bad = false;

  // Called before a group whose largest entry is vm > lim, or NaN. low: up to there an
  // entry (a finite mask, say) makes no reference; it weighs nothing beside ordinary entries.
  __device__ __forceinline__ void move(float vm, float low) {
    if (!(vm < INFINITY)) {  // NaN or +inf
      bad = true;
      return;
    }
    if (vm <= low) return;
    const float nc = -vm * kLog2e;
    if (lim != -INFINITY) {
      float old, unused;
      un2(c, old, unused);
      const float d = fmaxf(nc - old, -300.f), f = ex2(d);
      const uint64_t ff = pk2(f, f);
      T = mul2(fma2(S, pk2(d, d), T), ff);
      S = mul2(S, ff);
    }
    r = vm;
    c = pk2(nc, nc);
    lim = vm + kSlack;
  }
  // entries of at least the type's floor (p = 0 for the far ones)
  template <int N>
  __device__ __forceinline__ void add(const float* v, uint64_t L2) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t y = fma2(pk2(v[i], v[i + 1]), L2, c);
      float y0, y1;
      un2(y, y0, y1);
      const uint64_t p = pk2(ex2(y0), ex2(y1));
      S = add2(S, p);
      T = fma2(p, y, T);
    }
  }
};

// The largest entry that makes no reference.
template <typename T>
__device__ __forceinline__ constexpr float low_of() {
  return Vec<T>::kFloor > -kFar ? Vec<T>::kFloor : -kFar;
}

// A vector's entries, those below the type's floor raised to it, so that their y
// stays finite: the weight is 0 beside any ordinary entry, and 0 * y stays 0.
template <typename T>
__device__ __forceinline__ void unpack_floored(const uint4& raw, float* f) {
  Vec<T>::unpack(make_uint4(Vec<T>::floor_word(raw.x), Vec<T>::floor_word(raw.y), Vec<T>::floor_word(raw.z),
                            Vec<T>::floor_word(raw.w)),
                 f);
}

// Does entry (v, i) come before the token (value t at index tok)?
__device__ __forceinline__ bool is_ahead(float v, int i, float t, int tok) {
  if (t != t) return v != v && i < tok;
  return !(v < t) && (v != t || i < tok);
}

__device__ __forceinline__ void push(Shared& sh, float x, int i) {
  const unsigned at = atomicAdd(&sh.count, 1u);
  if (at < kCap) sh.list[at] = key_of(x, i);
}

// One CTA's part of a row: vectors [v0, v1) of the aligned body, and for the
// first CTA the entries before and after the body.
template <typename T>
struct Part {
  const T* x;
  const uint4* body;
  int head, v0, v1, vocab, edges;  // edges: entries outside the body (0 except for the first CTA)
  __device__ __forceinline__ int edge_index(int e) const {
    return e < head ? e : vocab - (edges - e);
  }
};

// Entries of a vector (first index i) that come before a NaN or infinite token.
template <typename T>
__device__ __noinline__ unsigned ahead_one_by_one(uint4 raw, int i, float t, int tok) {
  float f[Vec<T>::kN];
  Vec<T>::unpack(raw, f);
  unsigned n = 0;
#pragma unroll
  for (int j = 0; j < Vec<T>::kN; ++j) n += is_ahead(f[j], i + j, t, tok);
  return n;
}

// Notes a vector that holds a candidate.
__device__ __forceinline__ void note(Shared& sh, int v) {
  const unsigned at = atomicAdd(&sh.noted, 1u);
  if (at < kCap) sh.vecs[at] = v;
}

// The set bits of a thread's marks: bit b of mark u is the vector first + u * apart + b * kThreads.
__device__ __forceinline__ void note_marks(Shared& sh, uint32_t (&marks)[4], int first, int apart) {
  const unsigned n = __popc(marks[0]) + __popc(marks[1]) + __popc(marks[2]) + __popc(marks[3]);
  if (n == 0) return;
  unsigned at = atomicAdd(&sh.noted, n);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    for (; marks[u] && at < kCap; ++at) {
      const int b = __ffs(marks[u]) - 1;
      marks[u] &= marks[u] - 1;
      sh.vecs[at] = first + u * apart + b * kThreads;
    }
    marks[u] = 0;
  }
}

// A lower bound of the k-th largest of the block's values (k <= 32) that at
// least k of them reach: the k-th largest of each warp's four largest. Only
// distinct values of a warp count, so ties lower it; NaN counts as +inf.
__device__ __forceinline__ float block_bound(Shared& sh, float m, int k) {
  static_assert(kWarps * 4 == 32, "one value a lane");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t o = order_of(m != m ? INFINITY : m);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, o);
    if (lane == 0) sh.four[warp * 4 + j] = best;
    if (o == best) o = 0;  // below every value
  }
  __syncthreads();
  const uint32_t mine = sh.four[lane];
  int reach = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) reach += sh.four[j] >= mine;
  const uint32_t kth = __reduce_max_sync(0xffffffffu, reach >= k ? mine : 0u);
  return kth <= order_of(-INFINITY) ? -INFINITY : value_of(kth);
}

// Every vector with an entry at or above thr is noted.
template <typename T>
__device__ __noinline__ void collect(Shared& sh, const Part<T>& p, float thr) {
  for (int v = p.v0 + threadIdx.x; v < p.v1; v += kThreads)
    if (!(Vec<T>::value(largest<T>(p.body[v])) < thr)) note(sh, v);
}

// The entries at or above thr of the first n noted vectors, and of the edges, go to the list.
template <typename T>
__device__ __noinline__ void expand(Shared& sh, const Part<T>& p, unsigned n, float thr) {
  constexpr int N = Vec<T>::kN;
  for (unsigned a = threadIdx.x; a < n; a += kThreads) {
    const int v = sh.vecs[a];
    float f[N];
    Vec<T>::unpack(p.body[v], f);
    unsigned hits = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) hits |= f[j] < thr ? 0u : 1u << j;
    unsigned at = atomicAdd(&sh.count, (unsigned)__popc(hits));
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (hits >> j & 1u) {
        if (at < kCap) sh.list[at] = key_of(f[j], p.head + v * N + j);
        ++at;
      }
  }
  if (threadIdx.x < p.edges) {
    const int i = p.edge_index(threadIdx.x);
    const float f = Vec<T>::one(p.x + i);
    if (!(f < thr)) push(sh, f, i);
  }
  __syncthreads();
}

// The top entries by one scan per entry: for rows in which more than the list
// holds tie for a place.
template <typename T>
__device__ __noinline__ void top_by_scans(Shared& sh, const Part<T>& p, int top) {
  constexpr int N = Vec<T>::kN;
  uint64_t last = ~0ull, mine = 0;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int v = p.v0 + threadIdx.x; v < p.v1; v += kThreads) {
      float f[N];
      Vec<T>::unpack(p.body[v], f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint64_t key = key_of(f[j], p.head + v * N + j);
        if (key < last && key > best) best = key;
      }
    }
    if (threadIdx.x < p.edges) {
      const int i = p.edge_index(threadIdx.x);
      const uint64_t key = key_of(Vec<T>::one(p.x + i), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t w = shfl_xor64(best, o);
      best = w > best ? w : best;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.run[threadIdx.x >> 5][0] = best;
    __syncthreads();
    last = 0;
    for (int w = 0; w < kWarps; ++w) last = sh.run[w][0] > last ? sh.run[w][0] : last;
    if ((threadIdx.x & 31) == k) mine = last;
    if (last == 0) break;  // the part has no more entries
  }
  if (threadIdx.x < 32) sh.top[threadIdx.x] = mine;
  __syncthreads();
}

// Sorts the list's entries into sh.top.
__device__ __forceinline__ void sort_list(Shared& sh, unsigned n) {
  uint64_t best = 0;
  for (unsigned b = (threadIdx.x >> 5) * 32; b < n; b += kThreads) {  // uniform for a warp
    const unsigned at = b + (threadIdx.x & 31);
    const uint64_t v = sort32(at < n ? sh.list[at] : 0ull);
    best = b < kThreads ? v : merge32(best, v);
  }
  block_merge(sh, best, kWarps);
}

// The least value above x (x not NaN or +inf).
__device__ __forceinline__ float next_up(float x) { return value_of(order_of(x) + 1); }

// Adds entries equal to tie, in index order, to a list of fewer than top
// entries above it until it holds top; the part has enough of them.
template <typename T>
__device__ __noinline__ void fill_ties(Shared& sh, const Part<T>& p, float tie, unsigned top) {
  constexpr int N = Vec<T>::kN, kChunk = 1024 / N;  // the list has room for a chunk of ties
  if (threadIdx.x < p.edges) {
    const int i = p.edge_index(threadIdx.x);
    const float f = Vec<T>::one(p.x + i);
    if (f == tie) push(sh, f, i);
  }
  for (int v0 = p.v0; v0 < p.v1; v0 += kChunk) {
    __syncthreads();
    if (sh.count >= top + p.edges) break;  // the edges may come after the body
    __syncthreads();
    const int v = v0 + threadIdx.x;
    if (threadIdx.x < kChunk && v < p.v1) {
      float f[N];
      Vec<T>::unpack(p.body[v], f);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (f[j] == tie) push(sh, f[j], p.head + v * N + j);
    }
  }
  __syncthreads();
  sort_list(sh, min(sh.count, (unsigned)kCap));
}

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  Stats o;
  o.m = fmaxf(a.m, b.m);
  o.rank = a.rank + b.rank;
  o.bad = a.bad | b.bad;
  const float da = a.m == -INFINITY ? -200.f : fmaxf(a.m - o.m, -200.f);
  const float db = b.m == -INFINITY ? -200.f : fmaxf(b.m - o.m, -200.f);
  const float fa = ex2(da * kLog2e), fb = ex2(db * kLog2e);
  o.s = a.s * fa + b.s * fb;
  o.t = (a.t + da * a.s) * fa + (b.t + db * b.s) * fb;
  return o;
}

__device__ __forceinline__ Stats stats_of(const Sums& s, unsigned ahead) {
  float s0, s1, t0, t1, c, unused;
  un2(s.S, s0, s1);
  un2(s.T, t0, t1);
  un2(s.c, c, unused);
  const bool none = s.lim == -INFINITY;
  // 2^y stands for 2^(y + rest): c is -r L without its residue
  const float rest = none ? 0.f : fmaf(-s.r, kLog2e, -c), f = ex2(rest), S = (s0 + s1) * f;
  return Stats{none ? -INFINITY : s.r, none ? 0.f : S, none ? 0.f : ((t0 + t1) * f + rest * S) * kLn2, ahead,
               (unsigned)s.bad};
}

// The block's statistics, in every thread: each thread's sums are taken to the
// block's reference, then added in a fixed order.
__device__ __forceinline__ Stats block_join(Shared& sh, const Stats& st) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t o = __reduce_max_sync(0xffffffffu, order_of(st.m));
  if (lane == 0) sh.maxes[warp] = o;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) o = max(o, sh.maxes[w]);
  Stats a;
  a.m = value_of(o);
  const float d = st.m == -INFINITY ? -200.f : fmaxf(st.m - a.m, -200.f), f = ex2(d * kLog2e);
  a.s = st.s * f;
  a.t = (st.t + d * st.s) * f;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, k);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, k);
  }
  a.rank = __reduce_add_sync(0xffffffffu, st.rank);
  a.bad = __any_sync(0xffffffffu, st.bad);
  if (lane == 0) sh.warp[warp] = a;
  __syncthreads();
  a = sh.warp[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    a.s += sh.warp[w].s;
    a.t += sh.warp[w].t;
    a.rank += sh.warp[w].rank;
    a.bad |= sh.warp[w].bad;
  }
  return a;
}

// The part's sums again, entry by entry, each less the maximum before it is
// scaled: for parts whose largest entry is not well above low_of() (entries up to
// there have not been counted) or is beyond kFar.
template <typename T>
__device__ __noinline__ Stats sum_one_by_one(Shared& sh, const Part<T>& p, unsigned ahead) {
  float m = -INFINITY, S = 0.f, E = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    const auto take = [&](float v) {
      if (v == -INFINITY) return;
      if (pass == 0) {
        m = fmaxf(m, v);
      } else {
        const float z = fmaxf(v - m, -200.f), w = ex2(z * kLog2e);
        S += w;
        E += w * z;
      }
    };
    for (int i = p.head + p.v0 * Vec<T>::kN + threadIdx.x; i < p.head + p.v1 * Vec<T>::kN; i += kThreads)
      take(Vec<T>::one(p.x + i));
    if (threadIdx.x < p.edges) take(Vec<T>::one(p.x + p.edge_index(threadIdx.x)));
  }
  return block_join(sh, Stats{m, S, E, ahead, 0u});
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
    logprobs_kernel(const T* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ tokens, int vocab,
                    int top, int parts, float* __restrict__ logprob, int64_t* __restrict__ rank,
                    float* __restrict__ entropy, int64_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  kernel_entry();
  constexpr int N = Vec<T>::kN;
  __shared__ Shared sh;
  const int row = blockIdx.x / parts, part = blockIdx.x - row * parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = logits + (int64_t)row * row_stride;
  const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int head = min(mis ? N - mis : 0, vocab);
  const int nvec = (vocab - head) / N;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  const int edges = part == 0 ? vocab - nvec * N : 0;  // < 2 N
  const int v0 = (int)((int64_t)nvec * part / parts), v1 = (int)((int64_t)nvec * (part + 1) / parts);

  const int64_t tk = tokens[row];
  const bool has = tk >= 0 && tk < vocab;
  const int tok = has ? (int)tk : 0;
  const float t = Vec<T>::one(x + tok);
  if (threadIdx.x == 0) {
    sh.count = sh.noted = 0;
    if (!has && tk != -1 && part == 0) atomicOr(&g_err_logprobs, (unsigned)kErrTokenId);
  }

  // A step takes four blocks of 256 vectors, one from each quarter of the part's
  // whole steps, so the first step samples all of it; the last step takes what is left.
  const int quarter = (v1 - v0) / (4 * kThreads);
  const uint64_t L2 = pk2(kLog2e, kLog2e);
  Sums s;
  unsigned ahead = 0;
  float thr = INFINITY;  // least entry that may be among the top ones
  const bool plain = has && t < INFINITY;  // not a NaN or +inf
  const uint32_t t_bits = Vec<T>::bound(t != t ? -INFINITY : t);
  // the ties before the token in its own vector
  if (plain && threadIdx.x < N && tok >= head + v0 * N && tok < head + v1 * N) {
    const int i = tok - (tok - head) % N + threadIdx.x;
    ahead = i < tok && Vec<T>::one(x + i) == t;
  }
  uint32_t marks[4] = {0u, 0u, 0u, 0u};  // vectors of this thread that reach thr
  uint32_t thr_bits = Vec<T>::bound(thr), lim_bits = Vec<T>::bound(-INFINITY);
  // four vectors whose largest entries are vm, before their sums: the reference and the rank
  const auto look = [&](const uint4 (&raw)[4], const uint32_t (&vm)[4], int first, int apart) {
    const uint32_t most = Vec<T>::larger(Vec<T>::larger(vm[0], vm[1]), Vec<T>::larger(vm[2], vm[3]));
    if (Vec<T>::reaches(most, lim_bits)) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float m = Vec<T>::value(vm[u]);
        if (!(m <= s.lim)) s.move(m, low_of<T>());
      }
      lim_bits = Vec<T>::bound(s.lim);
    }
    if (!has || !Vec<T>::reaches(most, t_bits)) return;
    const uint32_t after = Vec<T>::above(t_bits);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int v = first + u * apart, i = head + v * N;
      if (v >= v1) continue;
      if (plain)  // before the token ties count too, from its own vector on they do not
        ahead += Vec<T>::count(raw[u], i + N <= tok ? t_bits : after);
      else
        ahead += ahead_one_by_one<T>(raw[u], i, t, tok);
    }
  };
  const auto sum = [&](const uint4& raw) {
    float f[N];
    unpack_floored<T>(raw, f);
    s.template add<N>(f, L2);
  };
  const auto first_bound = [&](const uint32_t (&vm)[4]) {
    thr = block_bound(sh, Vec<T>::value(Vec<T>::larger(Vec<T>::larger(vm[0], vm[1]), Vec<T>::larger(vm[2], vm[3]))), top);
    thr_bits = Vec<T>::bound(thr);  // exact: an entry
  };
  uint4 raw[4];
  uint32_t vm[4];
  if (quarter > 0) {
    // a vector's registers take the next step's as soon as it is summed, so four
    // loads a thread are nearly always in flight
    const uint4* at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at[u] = body + v0 + u * quarter * kThreads + threadIdx.x;
      raw[u] = __ldcs(at[u]);
    }
    for (int step = 0; step < quarter; ++step) {
      const int vs = v0 + step * kThreads + threadIdx.x, b = step % 32;
      const bool more = step + 1 < quarter;
#pragma unroll
      for (int u = 0; u < 4; ++u) vm[u] = largest<T>(raw[u]);
      if (top > 0) {
        if (step == 0)
          first_bound(vm);
        else if (b == 0)
          note_marks(sh, marks, vs - 32 * kThreads, quarter * kThreads);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (Vec<T>::reaches(vm[u], thr_bits)) marks[u] |= 1u << b;
      }
      look(raw, vm, vs, quarter * kThreads);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        sum(raw[u]);
        at[u] += kThreads;
        if (more) raw[u] = __ldcs(at[u]);
      }
    }
    if (top > 0) note_marks(sh, marks, v0 + (quarter - 1) / 32 * 32 * kThreads + threadIdx.x, quarter * kThreads);
  }
  {
    const int vs = v0 + quarter * 4 * kThreads + threadIdx.x;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      raw[u] = vs + u * kThreads < v1 ? __ldcs(body + vs + u * kThreads)
                                      : make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
      vm[u] = largest<T>(raw[u]);
    }
    if (top > 0) {
      if (quarter == 0) first_bound(vm);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (Vec<T>::reaches(vm[u], thr_bits) && vs + u * kThreads < v1) note(sh, vs + u * kThreads);
    }
    look(raw, vm, vs, kThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u) sum(raw[u]);
  }
  const Part<T> p = {x, body, head, v0, v1, vocab, edges};
  if (threadIdx.x < edges) {
    const int i = p.edge_index(threadIdx.x);
    const float v = Vec<T>::one(x + i);
    if (!(v <= s.lim)) s.move(v, low_of<T>());
    const float f[2] = {fmaxf(v, Vec<T>::kFloor), Vec<T>::kFloor};
    if (s.lim != -INFINITY) s.add<2>(f, L2);
    if (has) ahead += is_ahead(v, i, t, tok);
  }

  // ------------------------------------------------------ join the sums
  Stats st = stats_of(s, ahead);
  st = block_join(sh, st);
  // 256 above low_of(), what has not been counted weighs under e^-256
  if (!st.bad && !(st.m >= low_of<T>() + 256.f && st.m <= kFar)) st = sum_one_by_one(sh, p, ahead);
  if (threadIdx.x == 0) sh.cta = st;

  // ------------------------------------------------- the part's top entries
  if (top > 0) {
    float tie = NAN;
    for (int tries = 0;; ++tries) {
      const unsigned noted = sh.noted;
      expand(sh, p, min(noted, (unsigned)kCap), thr);
      const unsigned n = sh.count;
      sort_list(sh, min(n, (unsigned)kCap));
      if (noted <= kCap && n <= kCap) {
        if (tie == tie && n < (unsigned)top) fill_ties(sh, p, tie, top);
        break;
      }
      // More candidates than the lists hold: raise the bound to the list's own
      // k-th largest and look again, or, when that is a tie, past the tie, to
      // fill up with its first entries. Rows that rise along their length and
      // so overflow each time go without the lists.
      const float next = value_of((uint32_t)(sh.top[top - 1] >> 32));
      __syncthreads();
      if (tries == 3 || !(thr < INFINITY) || next != next) {
        top_by_scans(sh, p, top);
        break;
      }
      tie = next > thr ? NAN : thr;
      thr = next > thr ? next : next_up(thr);
      if (threadIdx.x == 0) sh.count = sh.noted = 0;
      __syncthreads();
      collect(sh, p, thr);
      __syncthreads();
    }
  } else {
    __syncthreads();
  }

  // -------------------------------------------------------- join the cluster
  if (parts > 1) {
    tc::cluster_sync_all();
    if (part == 0) {
      if (warp < parts) {
        const uint32_t top_at = tc::map_to_rank(smem_u32(&sh.top[lane]), warp);
        uint64_t v;
        asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(top_at) : "memory");
        sh.run[warp][lane] = v;
        if (lane < (int)(sizeof(Stats) / 4)) {
          const uint32_t at = tc::map_to_rank(smem_u32(reinterpret_cast<uint32_t*>(&sh.cta) + lane), warp);
          uint32_t w;
          asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
          reinterpret_cast<uint32_t*>(&sh.warp[warp])[lane] = w;
        }
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        Stats a = sh.warp[0];
        for (int c = 1; c < parts; ++c) a = join(a, sh.warp[c]);
        sh.cta = a;
      }
      const uint64_t v = warp < parts ? sh.run[warp][lane] : 0;
      __syncthreads();
      block_merge(sh, v, parts);
    }
    tc::cluster_sync_all();  // the other CTAs' shared memory is read until here
    if (part != 0) return;
  }
  if (warp == 0) {
    const Stats a = sh.cta;
    const float lse = logf(a.s);
    const auto lp_of = [&](float x) { return a.bad ? NAN : x == -INFINITY ? -INFINITY : (x - a.m) - lse; };
    if (lane == 0) {
      logprob[row] = has ? lp_of(t) : 0.f;
      rank[row] = has ? (int64_t)a.rank : -1;
      entropy[row] = a.bad ? NAN : a.m == -INFINITY ? 0.f : lse - a.t / a.s;
    }
    if (lane < top) {
      const uint64_t k = sh.top[lane];
      top_ids[(int64_t)row * top + lane] = 0x7fffffff - (int)(uint32_t)k;
      top_lp[(int64_t)row * top + lane] = lp_of(value_of((uint32_t)(k >> 32)));
    }
  }
}

// CTAs per row (1, 2, 4 or 8, the portable cluster sizes). More parts shorten
// the stream of a row but repeat its fixed work, so eight only while each CTA has
// an SM, four up to two CTAs an SM, two up to four (at 151936 bf16 entries and 20
// alternatives, us for 1/2/4/8 parts: 16 rows 22/16/12/11, 74 rows 24/18/17/23,
// 148 rows 30/23/29/38, 256 rows 36/31/38/56, 400 rows 41/47/55/83), and only
// while a part keeps a block of vectors.
int parts_for(int rows, int vectors) {
  const int64_t sms = device_sm_count();
  int parts = (int64_t)rows * 8 <= sms ? 8 : (int64_t)rows * 4 <= 2 * sms ? 4 : (int64_t)rows * 2 <= 4 * sms ? 2 : 1;
  while (parts > 1 && vectors / parts < kThreads) parts /= 2;
  return parts;
}

template <typename T>
int launch(const void* logits, int64_t row_stride, const int64_t* tokens, int rows, int vocab, int top, float* logprob,
           int64_t* rank, float* entropy, int64_t* top_ids, float* top_lp, cudaStream_t st) {
  const int parts = parts_for(rows, vocab / Vec<T>::kN);
  if ((int64_t)rows * parts > INT32_MAX) return set_error(kUnsupported, "kvb_token_logprobs: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * parts);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  attr[n].id = cudaLaunchAttributeClusterDimension;
  attr[n].val.clusterDim.x = (unsigned)parts;
  attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
  ++n;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cuda_status(cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, (const T*)logits, row_stride, tokens, vocab, top,
                                        parts, logprob, rank, entropy, top_ids, top_lp),
                     "kvb_token_logprobs launch");
}

}  // namespace
}  // namespace kvb

using namespace kvb;

extern "C" int kvb_token_logprobs(const void* logits, int dtype, int64_t row_stride, const int64_t* tokens, int rows,
                                  int vocab, int top_k, float* logprobs, int64_t* ranks, float* entropy,
                                  int64_t* top_ids, float* top_logprobs, void* stream) {
  if (rows < 0 || vocab <= 0 || vocab > (1 << 30) || row_stride < vocab)
    return set_error(kInvalid, "kvb_token_logprobs: bad sizes");
  if (dtype < 0 || dtype > 2) return set_error(kInvalid, "kvb_token_logprobs: unknown dtype %d", dtype);
  if (top_k < 0 || top_k > kMaxTop || top_k > vocab)
    return set_error(kUnsupported, "kvb_token_logprobs: top_k must be at most 32 and at most the vocabulary");
  if (rows == 0) return kOk;
  if (!logits || !tokens || !logprobs || !ranks || !entropy || (top_k && (!top_ids || !top_logprobs)))
    return set_error(kInvalid, "kvb_token_logprobs: NULL pointer");
  if ((uintptr_t)logits & (dtype == 2 ? 3 : 1)) return set_error(kInvalid, "kvb_token_logprobs: misaligned logits");
  const cudaStream_t st = (cudaStream_t)stream;
  if (dtype == 0)
    return launch<bf16>(logits, row_stride, tokens, rows, vocab, top_k, logprobs, ranks, entropy, top_ids, top_logprobs, st);
  if (dtype == 1)
    return launch<__half>(logits, row_stride, tokens, rows, vocab, top_k, logprobs, ranks, entropy, top_ids, top_logprobs, st);
  return launch<float>(logits, row_stride, tokens, rows, vocab, top_k, logprobs, ranks, entropy, top_ids, top_logprobs, st);
}
