// Log probabilities of given tokens, their ranks, each row's entropy and its
// most likely alternatives, from the logits.
//
// With m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):
//   logprob_i = (x_i - m) - log S,   entropy = log S - T / S
// (both terms of the entropy are non-negative, so nothing cancels). An entry of
// -inf has probability 0 and adds 0 to both sums; a row of only -inf has
// logprob -inf and entropy 0. A row with a NaN or +inf has NaN for each.
// Order of the entries: higher logit first, NaN above everything, the lower
// index on ties (-0 equals +0); rank counts the entries before the token.
#include <cuda_fp16.h>

#include "common.cuh"
#include "../../include/kavor_b200.h"

KVB_DEFINE_ERROR_WORD(logprobs)

namespace kvb {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }

// Whole number whose order is the order of the logits: NaN highest.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Entries in order: larger is earlier. Distinct for every index.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  return (uint64_t)order_of(x) << 32 | (uint32_t)(0x7fffffff - i);
}

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, Op op, T* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = op(v, sm[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    logprobs_kernel(const T* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ tokens, int vocab,
                    int top, float* __restrict__ logprob, int64_t* __restrict__ rank, float* __restrict__ entropy,
                    int64_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  kernel_entry();
  __shared__ uint64_t sm_u[kThreads / 32];
  __shared__ float sm_f[kThreads / 32];
  const T* x = logits + (int64_t)blockIdx.x * row_stride;
  const auto add = [](float a, float b) { return a + b; };
  const auto umax = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
  const auto uadd = [](uint64_t a, uint64_t b) { return a + b; };
  const int64_t tok = tokens[blockIdx.x];
  const bool has = tok >= 0 && tok < vocab;
  if (!has && tok != -1 && threadIdx.x == 0) atomicOr(&g_err_logprobs, (unsigned)kErrTokenId);
  const float xt = has ? as_float(x[tok]) : 0.f;
  const uint64_t kt = has ? key_of(xt, (int)tok) : ~0ull;
  float m = -INFINITY;
  uint64_t ahead = 0, best = 0;
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    const float v = as_float(x[i]);
    m = v != v || m != m ? NAN : fmaxf(m, v);
    const uint64_t k = key_of(v, i);
    best = k > best ? k : best;
    ahead += k > kt;
  }
  m = block_reduce(m, [](float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); }, sm_f);
  ahead = block_reduce(ahead, uadd, sm_u);
  const float ref = m == -INFINITY ? 0.f : m;
  float S = 0.f, E = 0.f;
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    const float z = as_float(x[i]) - ref;
    const float p = expf(z);
    S += p;
    E += p == 0.f ? 0.f : p * z;
  }
  S = block_reduce(S, add, sm_f);
  E = block_reduce(E, add, sm_f);
  const float lse = logf(S);
  if (threadIdx.x == 0) {
    logprob[blockIdx.x] = has ? (xt == -INFINITY && m == m && m != INFINITY ? -INFINITY : xt - ref - lse) : 0.f;
    rank[blockIdx.x] = has ? (int64_t)ahead : -1;
    entropy[blockIdx.x] = m == -INFINITY ? 0.f : lse - E / S;
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < top; ++j) {
    if (j > 0) {
      best = 0;
      for (int i = threadIdx.x; i < vocab; i += kThreads) {
        const uint64_t k = key_of(as_float(x[i]), i);
        if (k < last && k > best) best = k;
      }
    }
    last = block_reduce(best, umax, sm_u);
    if (threadIdx.x == 0) {
      const int id = 0x7fffffff - (int)(uint32_t)last;
      const float v = as_float(x[id]);
      top_ids[(int64_t)blockIdx.x * top + j] = id;
      top_lp[(int64_t)blockIdx.x * top + j] = v == -INFINITY && m == m && m != INFINITY ? -INFINITY : v - ref - lse;
    }
  }
}

template <typename T>
int launch(const void* logits, int64_t row_stride, const int64_t* tokens, int rows, int vocab, int top, float* logprob,
           int64_t* rank, float* entropy, int64_t* top_ids, float* top_lp, cudaStream_t st) {
  return cuda_status(launch_kernel(logprobs_kernel<T>, dim3(rows), dim3(kThreads), 0, st, (const T*)logits, row_stride,
                                   tokens, vocab, top, logprob, rank, entropy, top_ids, top_lp),
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
