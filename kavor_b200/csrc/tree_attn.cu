// Attention of drafted tokens over the paged KV cache (bf16 or e4m3 pages).
//
// Sequence b has context_lens[b] tokens in the cache; the last T_b of them are
// the nodes of its draft (T_b = cu_seqlens_q[b+1] - cu_seqlens_q[b] query
// rows). Node i sees every token before the draft and the nodes its mask bits
// name (with no mask: nodes 0..i, a chain). One node that sees itself is
// ordinary decode. For query head h of kv head h / G:
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j,  0 when nothing is seen.
// The e4m3 cache holds k_j = 2^a_j kq_j and v_j = 2^b_j vq_j; with
// x_j = scale * log2(e) * 2^a_j (q_i . kq_j) + b_j the weights 2^(x_j - max x)
// are at most 1 and multiply vq_j directly, and the softmax's own sum is
// sum_j 2^(x_j - max x) 2^(-b_j): both scales cost one FMA each.
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "common.cuh"
#include "../../include/kavor_b200.h"

KVB_DEFINE_ERROR_WORD(tree)

#include "tree_plan.cuh"

namespace kvb {
namespace {

using tree::Args;
using tree::kHD;
using tree::Walk;

// ------------------------------------------------------------- warp-MMA kernel
// 16 query rows (nodes x query heads of one kv head) per unit, 64-token tiles
// staged by TMA; each of four consumer warps takes 16 tokens of a tile.
constexpr int kRows = 16;
constexpr int kTile = 64;
constexpr int kWarps = 4;
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kScratchStride = kHD + 4;  // fp32 row of the warp merge, padded against bank conflicts

template <bool kFp8>
struct Cfg {
  static constexpr int kKV = kTile * kHD * (kFp8 ? 1 : 2);  // bytes of a K (or V) tile
  static constexpr int kStage = 2 * kKV;
  static constexpr int kStages = kFp8 ? 5 : 3;
  static constexpr int kSmem = kStages * kStage + kRows * kScratchStride * 4 + 1024;
};

__device__ __forceinline__ uint32_t swz_bf16(uint32_t base, int row, int chunk) {
  return base + (chunk >> 3) * (kTile * 128) + row * 128 + ((((chunk & 7) ^ (row & 7))) << 4);
}
__device__ __forceinline__ uint32_t swz_fp8(uint32_t base, int row, int chunk) {
  return base + row * 128 + ((chunk ^ (row & 7)) << 4);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two e4m3 bytes -> two halves (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
  return r;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

template <bool kFp8>
__global__ void __launch_bounds__(kThreads, 2)
    tree_warp_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ Args a) {
  using C = Cfg<kFp8>;
  kernel_entry();
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::kStages];
  __shared__ __align__(8) uint64_t empty_bar[C::kStages];
  __shared__ __align__(16) uint8_t scales[C::kStages][2][kTile];
  __shared__ float mw[kWarps][kRows], lw[kWarps][kRows];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scratch = reinterpret_cast<float*>(smem + C::kStages * C::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), kWarps);
    }
    fence_barrier_init();
  }
  const tree::Start start = tree::find_start<kThreads>(a, blockIdx.x);  // synchronises the block
  Walk w(a, start);

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
      const uint64_t pol = l2_evict_first_policy();
      uint32_t it = 0;
      bool ok = true;
      while (ok && w.next(a)) {
        int col = -1, blk = 0;
        bool bad = false;
        for (int j = 0; j < w.n; ++j, ++it) {
          const int s = it % C::kStages;
          if (it >= C::kStages && !mbar_wait(smem_u32(&empty_bar[s]), (it / C::kStages - 1) & 1, &g_err_tree)) {
            ok = false;
            break;
          }
          const int tok = (w.t0 + j) * kTile;
          if (tok / a.block_size != col) {
            col = tok / a.block_size;
            blk = a.tables[(int64_t)w.b * a.bt_stride + col];  // col < max_blocks: the length is cut to the table
            bad = blk < 0 || blk >= a.num_blocks;
            if (bad) {
              atomicOr(&g_err_tree, (unsigned)kErrBlockTable);
              blk = a.num_blocks;  // out of the tensor map: TMA fills zeros
            }
          }
          const int off = tok - col * a.block_size;
          const uint32_t st = smem_u32(smem + s * C::kStage);
          const uint32_t fb = smem_u32(&full_bar[s]);
          if (kFp8 && bad) {  // a block outside the pool reads zeros, of scale 1
            for (int i = 0; i < 2 * kTile / 4; ++i) reinterpret_cast<uint32_t*>(&scales[s][0][0])[i] = 0x7f7f7f7fu;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before a later copy into the same bytes
          }
          mbar_arrive_expect_tx(fb, C::kStage + (kFp8 && !bad ? 2 * kTile : 0));
          tma_load_4d(st, &kmap, 0, w.h, off, blk, fb, pol);
          if constexpr (!kFp8) tma_load_4d(st + C::kKV / 2, &kmap, 64, w.h, off, blk, fb, pol);
          tma_load_4d(st + C::kKV, &vmap, 0, w.h, off, blk, fb, pol);
          if constexpr (!kFp8) tma_load_4d(st + C::kKV + C::kKV / 2, &vmap, 64, w.h, off, blk, fb, pol);
          if (kFp8 && !bad) {
            const int64_t so = blk * a.scale_stride + (int64_t)w.h * a.block_size + off;
            bulk_load(smem_u32(&scales[s][0][0]), a.ks + so, kTile, fb);
            bulk_load(smem_u32(&scales[s][1][0]), a.vs + so, kTile, fb);
          }
        }
      }
      // no copy may outlive the CTA: wait (bounded) for the last phase of every stage
      for (uint32_t i = it < C::kStages ? 0 : it - C::kStages; i < it; ++i)
        mbar_wait(smem_u32(&full_bar[i % C::kStages]), (i / C::kStages) & 1, &g_err_tree);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int r = lane >> 2, j4 = lane & 3;  // rows r and r + 8, column group of the MMA fragments
  const int tok0 = warp * 16;
  uint32_t it = 0;
  bool ok = true;
  while (w.next(a)) {
    const int base = w.s.len - w.s.nodes;  // position of node 0 (negative: earlier nodes are not in the cache)
    int node[2], qrow[2];
    float rscale[2];
    uint32_t qa[8][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int R = w.rb * kRows + r + i * 8;
      node[i] = R / a.group;
      const bool in = node[i] < w.s.nodes;
      qrow[i] = w.s.q0 + (in ? node[i] : 0);
      const bf16* qp = a.q + (int64_t)qrow[i] * a.q_st + (int64_t)(w.h * a.group + (in ? R - node[i] * a.group : 0)) * a.q_sh;
      if constexpr (kFp8) {
        // the row over a power of two as halves: exact to 2^-25 of its largest
        // finite value, which is brought to [1, 2)
        uint2 raw[8];
        uint32_t mx = 0;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          raw[ks] = in ? *reinterpret_cast<const uint2*>(qp + ks * 16 + j4 * 4) : make_uint2(0u, 0u);
          const uint32_t x = raw[ks].x & 0x7fff7fffu, y = raw[ks].y & 0x7fff7fffu;
          mx = __vmaxu2(mx, __vmaxu2(x & ~__vcmpgtu2(x, 0x7f7f7f7fu), y & ~__vcmpgtu2(y, 0x7f7f7f7fu)));
        }
        mx = max(mx & 0xffffu, mx >> 16);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = min(max((int)(mx >> 7) - 127, -100), 100);
        const float inv = pow2(-e);
        rscale[i] = a.scale_log2 * pow2(e);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].x));
          const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].y));
          qa[ks][i] = pack_half(x.x * inv, x.y * inv);
          qa[ks][2 + i] = pack_half(y.x * inv, y.y * inv);
        }
      } else {
        rscale[i] = a.scale_log2;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          qa[ks][i] = in ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + j4 * 2) : 0u;
          qa[ks][2 + i] = in ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + j4 * 2 + 8) : 0u;
        }
      }
    }
    float o[16][4];
#pragma unroll
    for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

    for (int jt = 0; jt < w.n && ok; ++jt, ++it) {
      const int s = it % C::kStages;
      if (!mbar_wait(smem_u32(&full_bar[s]), (it / C::kStages) & 1, &g_err_tree)) {
        ok = false;
        break;
      }
      const uint32_t kb = smem_u32(smem + s * C::kStage), vb = kb + C::kKV;
      const int p0 = (w.t0 + jt) * kTile + tok0;  // position of this warp's first token
      bool odd_v = false;                          // a node's V row holds a value that is not finite
      if (p0 + 16 > base) {
        // The warp's tokens reach into the draft or past the context. Rows past
        // the context hold stale bytes (possibly NaN): zero them, since a zero
        // weight does not cancel NaN. Drafted rows may be hidden from some of
        // the query rows: look for values that a zero weight would not cancel.
        for (int idx = lane; idx < 16 * (kFp8 ? 8 : 16); idx += 32) {
          const int row = kFp8 ? idx >> 3 : idx >> 4, chunk = kFp8 ? idx & 7 : idx & 15;
          const uint32_t ad = kFp8 ? swz_fp8(vb, tok0 + row, chunk) : swz_bf16(vb, tok0 + row, chunk);
          if (p0 + row >= w.s.len) {
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ad), "r"(0u) : "memory");
          } else if (p0 + row >= base) {
            uint32_t x[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                         : "r"(ad));
#pragma unroll
            for (int i = 0; i < 4; ++i)
              odd_v |= kFp8 ? __vcmpeq4(x[i] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0
                            : __vcmpeq2(x[i] & 0x7f807f80u, 0x7f807f80u) != 0;
          }
        }
        odd_v = __any_sync(0xffffffffu, odd_v);
      }

      float sc[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
      const int mi = lane >> 3;
      if constexpr (kFp8) {
        // k-step ks covers 16 dims; lane j4 holds dims 4 j4 .. 4 j4 + 3 of it,
        // for Q and K alike (any order of the dims gives the same sum)
#pragma unroll
        for (int kp = 0; kp < 4; ++kp) {
          uint32_t b[4];
          ldmatrix_x4(swz_fp8(kb, tok0 + (lane & 7) + ((mi & 1) << 3), kp * 2 + (mi >> 1)), b[0], b[1], b[2], b[3]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mma_f16_16816(sc[q & 1], qa[kp * 2 + (q >> 1)], e4m3x2_to_half2(b[q]), e4m3x2_to_half2(b[q] >> 16));
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4(swz_bf16(kb, tok0 + (lane & 7) + ((mi >> 1) << 3), ks * 2 + (mi & 1)), b0, b1, b2, b3);
          mma_bf16_16816(sc[0], qa[ks], b0, b1);
          mma_bf16_16816(sc[1], qa[ks], b2, b3);
        }
      }

      float ev[2][2], inv_v[2][2];  // V exponents of this lane's four tokens
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int t = tok0 + j * 8 + j4 * 2 + e;
          if constexpr (kFp8) {
            const int kc = scales[s][0][t], vc = scales[s][1][t];
            const float ksc = __uint_as_float((uint32_t)kc << 23);
            ev[j][e] = (float)(vc - 127);
            inv_v[j][e] = __uint_as_float((uint32_t)(254 - vc) << 23);
            sc[j][e] = fmaf(sc[j][e], rscale[0] * ksc, ev[j][e]);
            sc[j][2 + e] = fmaf(sc[j][2 + e], rscale[1] * ksc, ev[j][e]);
          } else {
            inv_v[j][e] = 1.f;
            sc[j][e] *= rscale[0];
            sc[j][2 + e] *= rscale[1];
          }
        }
      uint32_t hidden = 0;  // bit j * 4 + half * 2 + e: that score is masked
      if (p0 + 16 > base) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int pos = p0 + j * 8 + j4 * 2 + e;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const bool seen = pos < base || (pos < w.s.len && tree::sees(a, qrow[i], node[i], pos - base));
              if (!seen) {
                sc[j][i * 2 + e] = -INFINITY;
                hidden |= 1u << (j * 4 + i * 2 + e);
              }
            }
          }
      }
      float p[2][4], corr[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(fmaxf(sc[0][2 * i], sc[0][2 * i + 1]), fmaxf(sc[1][2 * i], sc[1][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run[i], mx);
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        corr[i] = exp2f(m_run[i] - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = exp2f(sc[j][2 * i + e] - ref);
            p[j][2 * i + e] = x;
            // a masked weight is 0 whatever scale byte stands beside it
            sum += kFp8 ? (x == 0.f ? 0.f : x * inv_v[j][e]) : x;
          }
        l_run[i] = l_run[i] * corr[i] + sum;
        m_run[i] = m_new;
      }
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        o[n][0] *= corr[0];
        o[n][1] *= corr[0];
        o[n][2] *= corr[1];
        o[n][3] *= corr[1];
      }
      if (!odd_v) {
        // P is rounded to the type of the V operand: bf16, or half (2^-12) for e4m3
        const uint32_t pa[4] = {kFp8 ? pack_half(p[0][0], p[0][1]) : pack_bf16(p[0][0], p[0][1]),
                                kFp8 ? pack_half(p[0][2], p[0][3]) : pack_bf16(p[0][2], p[0][3]),
                                kFp8 ? pack_half(p[1][0], p[1][1]) : pack_bf16(p[1][0], p[1][1]),
                                kFp8 ? pack_half(p[1][2], p[1][3]) : pack_bf16(p[1][2], p[1][3])};
        if constexpr (kFp8) {
          // A transposed 8x8 of 16-bit elements gives a lane two tokens of a
          // pair of dims; a byte permutation pairs the tokens of each dim.
          // Accumulator 2c holds the even dims of 16-dim chunk c, 2c+1 the odd.
#pragma unroll
          for (int cp = 0; cp < 4; ++cp) {
            uint32_t b[4];
            ldmatrix_x4_trans(swz_fp8(vb, tok0 + (lane & 7) + ((mi & 1) << 3), cp * 2 + (mi >> 1)), b[0], b[1], b[2],
                              b[3]);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const uint32_t lo = __byte_perm(b[2 * q], 0, 0x3120), hi = __byte_perm(b[2 * q + 1], 0, 0x3120);
              mma_f16_16816(o[4 * cp + 2 * q], pa, e4m3x2_to_half2(lo), e4m3x2_to_half2(hi));
              mma_f16_16816(o[4 * cp + 2 * q + 1], pa, e4m3x2_to_half2(lo >> 16), e4m3x2_to_half2(hi >> 16));
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4_trans(swz_bf16(vb, tok0 + (lane & 7) + ((mi & 1) << 3), 2 * i + (mi >> 1)), b0, b1, b2, b3);
            mma_bf16_16816(o[2 * i], pa, b0, b1);
            mma_bf16_16816(o[2 * i + 1], pa, b2, b3);
          }
        }
      } else {
        // a drafted V row that is not finite: add only what each row sees, token
        // by token (rare, so it is written for size)
#pragma unroll 1
        for (int t = 0; t < 16; ++t) {
          const int src = (lane & ~3) | ((t & 7) >> 1), jj = t >> 3, e = t & 1;
          float pt[2];
          bool see[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float mine = jj ? (e ? p[1][2 * i + 1] : p[1][2 * i]) : (e ? p[0][2 * i + 1] : p[0][2 * i]);
            // every lane of the quad offers its own value for (jj, e); take the owner's
            pt[i] = __shfl_sync(0xffffffffu, mine, src);
            see[i] = !((__shfl_sync(0xffffffffu, hidden, src) >> (jj * 4 + i * 2 + e)) & 1u);
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if constexpr (kFp8) {
              const uint32_t x = lds32(swz_fp8(vb, tok0 + t, c) + j4 * 4);
#pragma unroll
              for (int d = 0; d < 4; ++d) {
                const uint32_t h2 = e4m3x2_to_half2(x >> (8 * d) & 0xffu);
                const float v = __low2float(*reinterpret_cast<const __half2*>(&h2));
                float* acc = o[2 * c + (d & 1)];
                if (see[0]) acc[d >> 1] += pt[0] * v;
                if (see[1]) acc[2 + (d >> 1)] += pt[1] * v;
              }
            } else {
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const uint32_t x = lds32(swz_bf16(vb, tok0 + t, 2 * c + hf) + j4 * 4);
                const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
                float* acc = o[2 * c + hf];
                if (see[0]) acc[0] += pt[0] * v.x, acc[1] += pt[0] * v.y;
                if (see[1]) acc[2] += pt[1] * v.x, acc[3] += pt[1] * v.y;
              }
            }
          }
        }
      }
      // order this warp's generic-proxy writes (tail zeroing) before the
      // producer's next async-proxy (TMA) write into the stage
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty_bar[s]));
    }

    // ------------------------------------------- join the four warps' tokens
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      if (j4 == 0) {
        mw[warp][r + i * 8] = m_run[i];
        lw[warp][r + i * 8] = l_run[i];
      }
    }
    named_bar_sync(1, kWarps * 32);
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float M = -INFINITY;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) M = fmaxf(M, mw[v][r + i * 8]);
      f[i] = m_run[i] == -INFINITY ? 0.f : exp2f(m_run[i] - M);
    }
#pragma unroll 1
    for (int turn = 0; turn < kWarps; ++turn) {
      if (warp == turn) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // both types: accumulators 2c and 2c+1 hold four dims of chunk c per row
            float v[4];
            int d[2];
            if constexpr (kFp8) {
              v[0] = o[2 * c][2 * i], v[1] = o[2 * c + 1][2 * i], v[2] = o[2 * c][2 * i + 1], v[3] = o[2 * c + 1][2 * i + 1];
              d[0] = c * 16 + j4 * 4, d[1] = d[0] + 2;
            } else {
              v[0] = o[2 * c][2 * i], v[1] = o[2 * c][2 * i + 1], v[2] = o[2 * c + 1][2 * i], v[3] = o[2 * c + 1][2 * i + 1];
              d[0] = c * 16 + j4 * 2, d[1] = d[0] + 8;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float2* at = reinterpret_cast<float2*>(scratch + (r + i * 8) * kScratchStride + d[x]);
              // a warp whose tokens were all masked contributes nothing (its rows are 0)
              float2 add = make_float2(v[2 * x] * f[i], v[2 * x + 1] * f[i]);
              if (turn > 0) {
                const float2 old = *at;
                add.x += old.x;
                add.y += old.y;
              }
              *at = add;
            }
          }
      }
      named_bar_sync(1, kWarps * 32);
    }
    const int row = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * 16;
    const int R = w.rb * kRows + row;
    const int nd = R / a.group;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) M = fmaxf(M, mw[v][row]);
#pragma unroll
    for (int v = 0; v < kWarps; ++v) L += mw[v][row] == -INFINITY ? 0.f : exp2f(mw[v][row] - M) * lw[v][row];
    if (!ok) M = -INFINITY, L = 0.f;
    const float* sp = scratch + row * kScratchStride + d0;
    if (nd < w.s.nodes) {
      if (w.whole()) {
        const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing seen: 0
        bf16* op = a.out + (int64_t)(w.s.q0 + nd) * a.o_st + (int64_t)(w.h * a.group + R - nd * a.group) * a.o_sh + d0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint4 y;
          y.x = pack_bf16(sp[8 * c] * inv, sp[8 * c + 1] * inv);
          y.y = pack_bf16(sp[8 * c + 2] * inv, sp[8 * c + 3] * inv);
          y.z = pack_bf16(sp[8 * c + 4] * inv, sp[8 * c + 5] * inv);
          y.w = pack_bf16(sp[8 * c + 6] * inv, sp[8 * c + 7] * inv);
          reinterpret_cast<uint4*>(op)[c] = y;
        }
      } else {
        const int64_t pr = ((int64_t)blockIdx.x * 2 + w.slot()) * kRows + row;
        float4* dst = reinterpret_cast<float4*>(a.part_o + pr * kHD + d0);
#pragma unroll
        for (int c = 0; c < 4; ++c) dst[c] = make_float4(sp[4 * c], sp[4 * c + 1], sp[4 * c + 2], sp[4 * c + 3]);
        if (d0 == 0) {
          a.part_m[pr] = M;
          a.part_l[pr] = L;
        }
      }
    }
    named_bar_sync(1, kWarps * 32);  // scratch and statistics are free again
  }
}

// ------------------------------------------------------------------- merge
// One warp per query row: joins the partials of a unit that was cut between
// CTAs, in CTA order, and writes zeros for a sequence with an empty context.
// Rows whose unit was whole have been written already.
constexpr int kMergeWarps = 8;

__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_kernel(const __grid_constant__ Args a) {
  kernel_entry();
  __shared__ int64_t s_first;
  const int b = blockIdx.y;
  const int per = (a.batch + kMergeWarps * 32 - 1) / (kMergeWarps * 32);
  const int b0 = min(threadIdx.x * per, a.batch), b1 = min(b0 + per, a.batch);
  int64_t mine = 0;
  for (int i = b0; i < b1; ++i) mine += tree::cost_of(a, tree::seq_of(a, i, false));
  int64_t total;
  int64_t at = tree::block_prefix<kMergeWarps * 32>(mine, &total);
  if (b0 <= b && b < b1) {
    for (int i = b0; i < b; ++i) at += tree::cost_of(a, tree::seq_of(a, i, false));
    s_first = at;
  }
  __syncthreads();
  const tree::Seq s = tree::seq_of(a, b, false);
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)s.nodes * a.hq;
  for (int64_t i = (int64_t)blockIdx.x * kMergeWarps + (threadIdx.x >> 5); i < rows;
       i += (int64_t)gridDim.x * kMergeWarps) {
    const int nd = (int)(i / a.hq), head = (int)(i - (int64_t)nd * a.hq);
    bf16* op = a.out + (int64_t)(s.q0 + nd) * a.o_st + (int64_t)head * a.o_sh + lane * 4;
    if (s.tiles == 0) {
      *reinterpret_cast<uint2*>(op) = make_uint2(0u, 0u);
      continue;
    }
    const int h = head / a.group;
    const int64_t R = (int64_t)nd * a.group + head - h * a.group;
    const int rb = (int)(R / a.rows), row = (int)(R - (int64_t)rb * a.rows);
    const int64_t lo = s_first + ((int64_t)h * s.blocks + rb) * s.tiles, hi = lo + s.tiles;
    int c = (int)(lo * a.parts / total);  // the part that holds tile lo
    while (c + 1 < a.parts && tree::part_begin(total, a.parts, c + 1) <= lo) ++c;
    while (c > 0 && tree::part_begin(total, a.parts, c) > lo) --c;
    if (tree::part_begin(total, a.parts, c + 1) >= hi) continue;  // whole
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int slot = 1;; ++c, slot = 0) {
      const int64_t pb = tree::part_begin(total, a.parts, c), pe = tree::part_begin(total, a.parts, c + 1);
      if (pb >= hi) break;
      if (pe > pb) {
        const int64_t pr = ((int64_t)c * 2 + slot) * a.rows + row;
        const float m = a.part_m[pr], l = a.part_l[pr];
        if (m != -INFINITY) {
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + pr * kHD + lane * 4);
          const float m_new = fmaxf(M, m);
          const float f0 = exp2f(M - m_new), f1 = exp2f(m - m_new);
          L = L * f0 + l * f1;
          acc.x = acc.x * f0 + x.x * f1;
          acc.y = acc.y * f0 + x.y * f1;
          acc.z = acc.z * f0 + x.z * f1;
          acc.w = acc.w * f0 + x.w * f1;
          M = m_new;
        }
      }
      if (c + 1 >= a.parts) break;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
}

// -------------------------------------------------------------------- host
int encode_pages(CUtensorMap* map, const void* base, bool fp8, int64_t num_blocks, int64_t block_stride_bytes,
                 int block_size, int hkv, int tile) {
  auto enc = tensor_map_encoder();
  if (!enc) return set_error(kNoEncoder, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t es = fp8 ? 1 : 2;
  const cuuint64_t dims[4] = {(cuuint64_t)kHD, (cuuint64_t)hkv, (cuuint64_t)block_size, (cuuint64_t)num_blocks};
  const cuuint64_t strides[3] = {kHD * es, (cuuint64_t)hkv * kHD * es, (cuuint64_t)block_stride_bytes};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / es), 1, (cuuint32_t)tile, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                   const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(kEncode, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
  return kOk;
}

size_t workspace_bytes(int parts, int rows) { return (size_t)parts * 2 * rows * (kHD + 2) * sizeof(float); }

template <bool kFp8>
int launch_warp(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "kvb_tree_attn: cudaGetDevice");
  if (dev >= 64 || !((done.load() >> dev) & 1ull)) {
    e = cudaFuncSetAttribute(tree_warp_kernel<kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<kFp8>::kSmem);
    if (e != cudaSuccess) return cuda_status(e, "kvb_tree_attn: shared memory attribute");
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  e = launch_kernel(tree_warp_kernel<kFp8>, dim3(a.parts), dim3(kThreads), Cfg<kFp8>::kSmem, st, km, vm, a);
  return cuda_status(e, "kvb_tree_attn launch");
}

}  // namespace
}  // namespace kvb

using namespace kvb;

extern "C" int kvb_tree_attn_workspace_size(int num_q_heads, int num_kv_heads, int max_seqlen_q, size_t* bytes) {
  if (!bytes) return set_error(kInvalid, "kvb_tree_attn_workspace_size: bytes is NULL");
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || max_seqlen_q < 0)
    return set_error(kInvalid, "kvb_tree_attn_workspace_size: bad sizes");
  *bytes = workspace_bytes(2 * device_sm_count(), kRows);
  return kOk;
}

extern "C" int kvb_tree_attn(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t total_q,
                             const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                             int64_t num_blocks, int64_t block_stride, int64_t scale_block_stride, int block_size,
                             const int32_t* block_tables, int64_t block_table_stride, int max_blocks_per_seq,
                             const int32_t* context_lens, const int32_t* cu_seqlens_q, int max_seqlen_q,
                             const int32_t* tree_mask, int64_t mask_stride, int mask_words, void* out,
                             int64_t out_stride_t, int64_t out_stride_h, int batch, int num_q_heads, int num_kv_heads,
                             int head_dim, float scale, void* workspace, size_t workspace_bytes_given, void* stream) {
  if (batch < 0 || total_q < 0 || total_q > INT32_MAX || num_q_heads <= 0 || num_kv_heads <= 0 ||
      num_q_heads % num_kv_heads || num_blocks <= 0 || num_blocks >= INT32_MAX || block_size <= 0 ||
      max_blocks_per_seq < 0 || max_seqlen_q < 0 || mask_words < 0)
    return set_error(kInvalid, "kvb_tree_attn: bad sizes");
  if (head_dim != kHD) return set_error(kUnsupported, "kvb_tree_attn: head_dim must be 128");
  if (block_size % 64) return set_error(kUnsupported, "kvb_tree_attn: block_size must be a multiple of 64");
  if (batch > 65535) return set_error(kUnsupported, "kvb_tree_attn: more than 65535 sequences");
  if ((int64_t)max_blocks_per_seq * block_size > INT32_MAX - 1024)
    return set_error(kUnsupported, "kvb_tree_attn: block tables of more than 2^31 tokens");
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return kOk;
  const bool fp8 = k_scale != nullptr;
  if (!q || !k_cache || !v_cache || !context_lens || !cu_seqlens_q || !out || (!block_tables && max_blocks_per_seq) ||
      (fp8 && !v_scale))
    return set_error(kInvalid, "kvb_tree_attn: NULL pointer");
  if (((uintptr_t)q & 15) || q_stride_t % 8 || q_stride_h % 8 || ((uintptr_t)out & 15) || out_stride_t % 8 ||
      out_stride_h % 8)
    return set_error(kInvalid, "kvb_tree_attn: query and output rows must be 16-byte aligned");
  const int64_t page = (int64_t)block_size * num_kv_heads * kHD;
  if (((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15) || block_stride % (fp8 ? 16 : 8) || block_stride < page)
    return set_error(kInvalid, "kvb_tree_attn: cache must be 16-byte aligned with a full block stride");
  if (fp8 && (((uintptr_t)k_scale & 15) || ((uintptr_t)v_scale & 15) || scale_block_stride % 16 ||
              scale_block_stride < (int64_t)block_size * num_kv_heads))
    return set_error(kInvalid, "kvb_tree_attn: scales must be 16-byte aligned with a full block stride");
  if (tree_mask && (mask_words == 0 || mask_stride < 0))
    return set_error(kInvalid, "kvb_tree_attn: a mask has at least one word a row and no negative stride");
  if (!(scale > 0.f) || scale > 1e30f) return set_error(kInvalid, "kvb_tree_attn: scale must be positive and finite");

  Args a = {};
  a.rows = kRows;
  a.tile = kTile;
  a.parts = 2 * device_sm_count();
  const size_t need = workspace_bytes(a.parts, a.rows);
  if (!workspace || workspace_bytes_given < need)
    return set_error(kWorkspace, "kvb_tree_attn: workspace of %zu bytes needed, %zu given", need,
                     workspace ? workspace_bytes_given : (size_t)0);
  if ((uintptr_t)workspace & 15) return set_error(kInvalid, "kvb_tree_attn: workspace alignment");
  a.q = (const bf16*)q;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.total_q = total_q;
  a.tables = block_tables;
  a.bt_stride = block_table_stride;
  a.max_blocks = max_blocks_per_seq;
  a.ctx = context_lens;
  a.cu_q = cu_seqlens_q;
  a.mask = (const uint32_t*)tree_mask;
  a.mask_stride = mask_stride;
  a.mask_words = mask_words;
  a.out = (bf16*)out;
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.ks = (const uint8_t*)k_scale;
  a.vs = (const uint8_t*)v_scale;
  a.scale_stride = scale_block_stride;
  a.batch = batch;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.num_blocks = (int)num_blocks;
  a.block_size = block_size;
  a.part_o = (float*)workspace;
  a.part_m = a.part_o + (size_t)a.parts * 2 * a.rows * kHD;
  a.part_l = a.part_m + (size_t)a.parts * 2 * a.rows;
  a.scale_log2 = scale * 1.4426950408889634f;

  CUtensorMap km, vm;
  const int64_t bytes = block_stride * (fp8 ? 1 : 2);
  int rc = encode_pages(&km, k_cache, fp8, num_blocks, bytes, block_size, num_kv_heads, a.tile);
  if (!rc) rc = encode_pages(&vm, v_cache, fp8, num_blocks, bytes, block_size, num_kv_heads, a.tile);
  if (!rc) rc = fp8 ? launch_warp<true>(km, vm, a, (cudaStream_t)stream) : launch_warp<false>(km, vm, a, (cudaStream_t)stream);
  if (rc) return rc;
  const int64_t mrows = ((int64_t)max_seqlen_q * num_q_heads + kMergeWarps - 1) / kMergeWarps;
  return cuda_status(launch_kernel(tree_merge_kernel, dim3((unsigned)(mrows < 4096 ? mrows : 4096), (unsigned)batch),
                                   dim3(kMergeWarps * 32), 0, (cudaStream_t)stream, a),
                     "kvb_tree_attn merge launch");
}
