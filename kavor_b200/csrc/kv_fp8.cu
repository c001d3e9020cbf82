// The paged KV cache in 8 bits: quantise on write, read back as bf16.
//
// A row (one token, one kv head, 128 values) is held as 128 e4m3 bytes and one
// e8m0 byte c that stands for the scale 2^(c - 127). With e the smallest whole
// number such that the row's largest finite magnitude is at most 448 * 2^e
// (448 is the largest e4m3 value; e is clamped to [-100, 120], 0 for a zero
// row), the held value is e4m3(x / 2^e), rounded to nearest even. A power of
// two costs a float format no precision (the relative error of a normal value
// is 2^-4 at any scale) and makes both directions exact: x / 2^e only changes
// the exponent, so the one rounding is the e4m3 one, and q * 2^e (4 significant
// bits) is a bf16 value again. Infinities are held as the row's largest value
// +-448 * 2^e, NaN as NaN; neither counts for the scale. (Values within 1/32 of the
// largest bf16 value round to 2^128, which a bf16 read gives as infinity.)
//
// Both kernels are bound by HBM (and, at a decode batch, by one launch): 8 lanes
// (write) or 16 (read) own one row, so a warp moves whole rows with full-width
// accesses and the row maximum takes three shuffles. Measured: 16384 tokens of 8
// heads written in 18.5 us (5.5 TB/s of rows, cache bytes and scales), 64 sequences of
// 100 to 4000 tokens read back in 152 us (5.3 TB/s).
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "../../include/kavor_b200.h"

KVB_DEFINE_ERROR_WORD(kv_fp8)

namespace kvb {
namespace {

constexpr int kHD = 128;
constexpr int kThreads = 256;
constexpr int kRowLanes = 16;
constexpr int kRowsPerBlock = kThreads / kRowLanes;
// The write gives a lane two 16-byte pieces of a row, 64 values apart: what is done
// once a row and lane is most of its instructions (16 lanes a row: 21.7 us, this 18.5
// for 16384 tokens of 8 heads).
constexpr int kStoreLanes = 8, kStoreRows = kThreads / kStoreLanes;

struct CacheRef {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;
  uint8_t* vs;
  int64_t num_blocks, block_stride, scale_stride;  // strides between blocks, bytes
  int block_size, hkv;
};

// n / d for 0 <= n < 2^31 by one multiplication: with 2^(s-1) < d <= 2^s and mul =
// ceil(2^(31+s) / d), n mul / 2^(31+s) exceeds n / d by less than n / 2^(31+s) <
// 2^-s <= 1 / d, so the whole parts agree. (The rows' and slots' divisions were a
// third of the write's instructions.)
struct Divisor {
  uint32_t mul;
  int shift;
  explicit Divisor(int d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    shift = 31 + s;
    mul = (uint32_t)(((1ull << shift) + (uint64_t)d - 1) / (uint64_t)d);
  }
  __device__ __forceinline__ int divide(int n) const { return (int)((uint64_t)(uint32_t)n * mul >> shift); }
};

// Largest magnitudes of 8 bf16 values of k (low half) and of v, infinities and NaN
// included: the largest finite ones where no infinity or NaN is among them.
__device__ __forceinline__ uint32_t max8_of_two(const uint4& k, const uint4& v) {
  constexpr uint32_t m = 0x7fff7fffu;
  const uint32_t a = __vmaxu2(__vmaxu2(k.x & m, k.y & m), __vmaxu2(k.z & m, k.w & m));
  const uint32_t b = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  return __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
}
// Largest finite magnitude of 8 bf16 values, as bf16 bits: for positive
// floats the order of the bits is the order of the values.
__device__ __forceinline__ uint32_t finite_max8(const uint4& r) {
  const uint32_t w[4] = {r.x & 0x7fff7fffu, r.y & 0x7fff7fffu, r.z & 0x7fff7fffu, r.w & 0x7fff7fffu};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & ~__vcmpgtu2(w[i], 0x7f7f7f7fu));
  return max(m & 0xffffu, m >> 16);
}

// Exponent e of the row's scale from its largest magnitude's bf16 bits:
// 1.m * 2^x <= 1.75 * 2^8 * 2^e, so e = x - 8, or x - 7 when 1.m > 1.75.
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
  if (bits == 0) return 0;
  const int x = (int)(bits >> 7) - 127;
  const int e = x - 8 + ((bits & 0x7fu) > 0x60u);
  return max(e, -100);
}

// bf16 pairs times 2^-e to four e4m3 bytes.
__device__ __forceinline__ uint32_t quantise4(uint32_t lo, uint32_t hi, float inv) {
  const float2 a = make_float2(__uint_as_float(lo << 16) * inv, __uint_as_float(lo & 0xffff0000u) * inv);
  const float2 b = make_float2(__uint_as_float(hi << 16) * inv, __uint_as_float(hi & 0xffff0000u) * inv);
  return __byte_perm(__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3),
                     __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3), 0x5410);
}
__device__ __forceinline__ uint2 quantise8(const uint4& r, int e) {
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  return make_uint2(quantise4(r.x, r.y, inv), quantise4(r.z, r.w, inv));
}

__global__ void __launch_bounds__(kThreads)
    store_kv_fp8_kernel(const bf16* __restrict__ key, int64_t k_st, int64_t k_sh, const bf16* __restrict__ value,
                        int64_t v_st, int64_t v_sh, CacheRef c, Divisor by_heads, Divisor by_block,
                        const int32_t* __restrict__ slots, int rows) {
  kernel_entry();
  const int64_t row = (int64_t)blockIdx.x * kStoreRows + threadIdx.x / kStoreLanes;
  const int lane = threadIdx.x % kStoreLanes;
  const int rr = row < rows ? (int)row : rows - 1;  // every lane takes part in the shuffles
  const int t = by_heads.divide(rr), h = rr - t * c.hkv;
  const int32_t slot = slots[t];
  const uint4* kp = reinterpret_cast<const uint4*>(key + t * k_st + h * k_sh) + lane;
  const uint4* vp = reinterpret_cast<const uint4*>(value + t * v_st + h * v_sh) + lane;
  const uint4 k0 = kp[0], k1 = kp[kStoreLanes], v0 = vp[0], v1 = vp[kStoreLanes];
  uint32_t mx = __vmaxu2(max8_of_two(k0, v0), max8_of_two(k1, v1));
#pragma unroll
  for (int o = kStoreLanes / 2; o > 0; o >>= 1) mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (__any_sync(0xffffffffu, (mx & 0xffffu) > 0x7f7fu || mx > 0x7f7fffffu)) {  // rare: an infinity or NaN in the warp's rows
    mx = max(finite_max8(k0), finite_max8(k1)) | max(finite_max8(v0), finite_max8(v1)) << 16;
#pragma unroll
    for (int o = kStoreLanes / 2; o > 0; o >>= 1) mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (row >= rows || slot == -1) return;
  if (slot < 0 || slot >= c.num_blocks * c.block_size) {
    if (lane == 0) atomicOr(&g_err_kv_fp8, (unsigned)kErrSlot);
    return;
  }
  const int64_t blk = by_block.divide(slot);
  const int off = slot - (int)blk * c.block_size;
  const int ek = scale_exponent(mx & 0xffffu), ev = scale_exponent(mx >> 16);
  const int64_t at = blk * c.block_stride + ((int64_t)off * c.hkv + h) * kHD;
  uint2* kd = reinterpret_cast<uint2*>(c.k + at) + lane;
  uint2* vd = reinterpret_cast<uint2*>(c.v + at) + lane;
  kd[0] = quantise8(k0, ek);
  kd[kStoreLanes] = quantise8(k1, ek);
  vd[0] = quantise8(v0, ev);
  vd[kStoreLanes] = quantise8(v1, ev);
  if (lane < 2) {
    const int64_t sat = blk * c.scale_stride + (int64_t)h * c.block_size + off;
    (lane == 0 ? c.ks : c.vs)[sat] = (uint8_t)((lane == 0 ? ek : ev) + 127);
  }
}

__device__ __forceinline__ uint4 dequantise8(uint2 q, float scale) {
  const uint32_t w[2] = {q.x, q.y};
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> ((i & 1) * 16)), __NV_E4M3);
    const float2 f = __half22float2(__half2(hr));
    out[i] = pack_bf16(f.x * scale, f.y * scale);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

constexpr int kLoadTokens = 32;  // flat tokens per CTA

__global__ void __launch_bounds__(kThreads)
    load_kv_fp8_kernel(CacheRef c, const int32_t* __restrict__ tables, int64_t bt_stride, int max_blocks,
                       const int32_t* __restrict__ cu, int batch, int total, bf16* __restrict__ ko, int64_t ko_st,
                       bf16* __restrict__ vo, int64_t vo_st) {
  kernel_entry();
  __shared__ int s_blk[kLoadTokens], s_off[kLoadTokens];
  const int t0 = blockIdx.x * kLoadTokens;
  // the sequence of the CTA's first token: how many sequences end at or before it
  int ended = 0;
  for (int i0 = 0; i0 < batch; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    ended += __syncthreads_count(i < batch && cu[i + 1] <= t0);
  }
  if (threadIdx.x < kLoadTokens) {
    const int t = t0 + threadIdx.x;
    int blk = -2, off = 0, b = ended;
    if (t < total) {
      while (b < batch && cu[b + 1] <= t) ++b;
      if (b < batch && t >= cu[b]) {  // rows past the last sequence are left as they are
        const int pos = t - cu[b];
        const int col = pos / c.block_size;
        off = pos - col * c.block_size;
        blk = col < max_blocks ? tables[(int64_t)b * bt_stride + col] : -1;
        if (blk < 0 || blk >= c.num_blocks) {
          atomicOr(&g_err_kv_fp8, (unsigned)kErrBlockTable);
          blk = -1;
        }
      }
    }
    s_blk[threadIdx.x] = blk;
    s_off[threadIdx.x] = off;
  }
  __syncthreads();
  const int lane = threadIdx.x % kRowLanes;
  for (int r = threadIdx.x / kRowLanes; r < kLoadTokens * c.hkv; r += kRowsPerBlock) {
    const int tt = r / c.hkv, h = r - tt * c.hkv;
    const int blk = s_blk[tt];
    if (blk == -2) continue;
    uint4 ky = make_uint4(0, 0, 0, 0), vy = ky;
    if (blk >= 0) {
      const int64_t at = blk * c.block_stride + ((int64_t)s_off[tt] * c.hkv + h) * kHD + lane * 8;
      const int64_t sat = blk * c.scale_stride + (int64_t)h * c.block_size + s_off[tt];
      const uint2 kq = *reinterpret_cast<const uint2*>(c.k + at);
      const uint2 vq = *reinterpret_cast<const uint2*>(c.v + at);
      ky = dequantise8(kq, __uint_as_float((uint32_t)c.ks[sat] << 23));
      vy = dequantise8(vq, __uint_as_float((uint32_t)c.vs[sat] << 23));
    }
    const int64_t t = t0 + tt;
    *reinterpret_cast<uint4*>(ko + t * ko_st + h * kHD + lane * 8) = ky;
    *reinterpret_cast<uint4*>(vo + t * vo_st + h * kHD + lane * 8) = vy;
  }
}

inline bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Checks shared by both entry points; fills the reference to the cache.
int cache_ref(CacheRef* c, const char* who, const void* k, const void* v, const void* ks, const void* vs,
              int64_t num_blocks, int64_t block_stride, int64_t scale_stride, int block_size, int hkv, int head_dim) {
  if (num_blocks < 0 || num_blocks >= INT32_MAX || block_size <= 0 || hkv <= 0)
    return set_error(kInvalid, "%s: bad sizes", who);
  if (head_dim != kHD) return set_error(kUnsupported, "%s: head_dim must be 128", who);
  if (!k || !v || !ks || !vs) return set_error(kInvalid, "%s: NULL pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16) || block_stride % 16)
    return set_error(kInvalid, "%s: the cache and its block stride must be 16-byte aligned", who);
  if (block_stride < (int64_t)block_size * hkv * kHD || scale_stride < (int64_t)block_size * hkv)
    return set_error(kInvalid, "%s: block stride smaller than one block", who);
  *c = CacheRef{(uint8_t*)k, (uint8_t*)v, (uint8_t*)ks, (uint8_t*)vs, num_blocks, block_stride, scale_stride,
                block_size, hkv};
  return kOk;
}

}  // namespace
}  // namespace kvb

using namespace kvb;

extern "C" int kvb_store_kv_fp8(const void* key, int64_t key_stride_t, int64_t key_stride_h, const void* value,
                                int64_t value_stride_t, int64_t value_stride_h, void* k_cache, void* v_cache,
                                void* k_scale, void* v_scale, int64_t num_blocks, int64_t block_stride,
                                int64_t scale_block_stride, int block_size, int num_kv_heads, int head_dim,
                                const int32_t* slot_mapping, int num_tokens, void* stream) {
  if (num_tokens < 0) return set_error(kInvalid, "kvb_store_kv_fp8: bad sizes");
  if (num_tokens == 0) return kOk;
  CacheRef c;
  int rc = cache_ref(&c, "kvb_store_kv_fp8", k_cache, v_cache, k_scale, v_scale, num_blocks, block_stride,
                     scale_block_stride, block_size, num_kv_heads, head_dim);
  if (rc) return rc;
  if (!key || !value || !slot_mapping) return set_error(kInvalid, "kvb_store_kv_fp8: NULL pointer");
  if (!aligned(key, 16) || !aligned(value, 16) || key_stride_t % 8 || key_stride_h % 8 || value_stride_t % 8 ||
      value_stride_h % 8)
    return set_error(kInvalid, "kvb_store_kv_fp8: key/value rows must be 16-byte aligned");
  const int64_t rows = (int64_t)num_tokens * num_kv_heads;
  if (rows > INT32_MAX) return set_error(kUnsupported, "kvb_store_kv_fp8: more than 2^31 rows");
  const int64_t grid = (rows + kStoreRows - 1) / kStoreRows;
  return cuda_status(launch_kernel(store_kv_fp8_kernel, dim3((unsigned)grid), dim3(kThreads), 0, (cudaStream_t)stream,
                                   (const bf16*)key, key_stride_t, key_stride_h, (const bf16*)value, value_stride_t,
                                   value_stride_h, c, Divisor(num_kv_heads), Divisor(block_size), slot_mapping, (int)rows),
                     "kvb_store_kv_fp8 launch");
}

extern "C" int kvb_load_kv_fp8(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                               int64_t num_blocks, int64_t block_stride, int64_t scale_block_stride, int block_size,
                               int num_kv_heads, int head_dim, const int32_t* block_tables,
                               int64_t block_table_stride, int max_blocks_per_seq, const int32_t* cu_seqlens_k,
                               int batch, int total_k, void* k_out, int64_t k_out_stride_t, void* v_out,
                               int64_t v_out_stride_t, void* stream) {
  if (batch < 0 || total_k < 0 || max_blocks_per_seq < 0) return set_error(kInvalid, "kvb_load_kv_fp8: bad sizes");
  if (batch == 0 || total_k == 0) return kOk;
  CacheRef c;
  int rc = cache_ref(&c, "kvb_load_kv_fp8", k_cache, v_cache, k_scale, v_scale, num_blocks, block_stride,
                     scale_block_stride, block_size, num_kv_heads, head_dim);
  if (rc) return rc;
  if (!block_tables || !cu_seqlens_k || !k_out || !v_out) return set_error(kInvalid, "kvb_load_kv_fp8: NULL pointer");
  const int64_t row = (int64_t)num_kv_heads * kHD;
  if (!aligned(k_out, 16) || !aligned(v_out, 16) || k_out_stride_t % 8 || v_out_stride_t % 8 || k_out_stride_t < row ||
      v_out_stride_t < row)
    return set_error(kInvalid, "kvb_load_kv_fp8: output rows must be 16-byte aligned and hold all heads");
  const int grid = (int)(((int64_t)total_k + kLoadTokens - 1) / kLoadTokens);
  return cuda_status(launch_kernel(load_kv_fp8_kernel, dim3(grid), dim3(kThreads), 0, (cudaStream_t)stream, c,
                                   block_tables, block_table_stride, max_blocks_per_seq, cu_seqlens_k, batch, total_k,
                                   (bf16*)k_out, k_out_stride_t, (bf16*)v_out, v_out_stride_t),
                     "kvb_load_kv_fp8 launch");
}
