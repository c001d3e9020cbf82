// Attention of drafted tokens over the paged KV cache (bf16 or e4m3 pages).
//
// Sequence b has context_lens[b] tokens in the cache; the last T_b of them are
// the nodes of its draft (T_b = cu_seqlens_q[b+1] - cu_seqlens_q[b] query
// rows). Node i sees every token before the draft and the nodes its mask bits
// name (with no mask: nodes 0..i, a chain). One node that sees itself is
// ordinary decode. For query head h of kv head h / G:
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j,  0 when nothing is seen.
// The e4m3 cache holds k_j = 2^a_j kq_j and v_j = 2^b_j vq_j. K's scale multiplies
// the score; V's goes into the weight where few query rows share a V (first kernel)
// and into V where many do (tree_attn_tc.cuh).
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "common.cuh"
#include "../../include/kavor_b200.h"

KVB_DEFINE_ERROR_WORD(tree)

#include "tcgen05.cuh"
#include "tree_plan.cuh"

namespace kvb {
namespace {

using tree::Args;
using tree::kHD;
using tree::Walk;

// ------------------------------------------------------------- warp-MMA kernel
// 8 NT query rows (nodes x query heads) of each of HP kv heads per unit, tiles of
// 64 KT / HP tokens staged by TMA; each of four consumer warps takes 16 KT tokens
// of one head. Tokens
// (then head dims) are the MMAs' 16-row side and query rows their 8-column side,
// S^T = K Q^T and O^T = V^T P^T, so a decode step's 4 to 8 query heads fill the
// instructions and K and V are converted once for all rows. e4m3 bytes become
// halves in registers (exact); two 8x8 register transposes turn the weights from
// S^T's layout to P^T's.
//
// Over e4m3 the weights are halves and carry V's scale: with s_j = scale log2(e) 2^a_j
// (q . kq_j) and a row's running reference m = max(s_j + b_j), vq_j is multiplied by
// 2^(s_j + b_j - m + 8). That is the row's share of the output, so what a half loses
// (steps of 2^-24) is 2^-33 of the largest share at most. The softmax's own sum is of
// 2^(s_j - m + 8) in 32 bits: taken from the weight, times 2^-b_j, it lost tokens whose
// share is small only because their V is. The weight is that term times 2^b_j (for 16
// rows a second exponential was slower: 16 rows over 256 x 1024 tokens 143 us, this 139).
// A row of V that holds nothing has the scale 2^0 and no share: it counts with kNothing
// for b_j, or one that draws the attention would push every other weight out of a half's
// range. Two rows go through each step together (a row at a time: 146 us). A reference
// can lie 2^220 above the one before it (a block of large rows of V after one of zeros)
// while the sum so far, up to 2^108 a token, still counts: it is scaled in two steps of
// half the way.
constexpr float kTop = 8.f;         // log2 of the largest weight over e4m3
constexpr float kNothing = -100.f;  // the least exponent a written row can have
constexpr int kWarps = 4;
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kScratchStride = kHD + 4;  // fp32 row of the warp merge, padded against bank conflicts

template <bool kFp8, int NT, int HP>
struct Cfg {
  static constexpr int kRows = 8 * NT;
  // e4m3 tiles hold twice the tokens: as many bytes a stage, and two chains of
  // MMAs a warp, whose softmax steps overlap
  static constexpr int KT = kFp8 ? 2 : 1;
  // A token's row of one e4m3 head is 128 bytes, num_kv_heads * 128 apart. One
  // head a unit left HBM at 5.1 TB/s (256 x 1024 tokens, 8 heads, loads alone):
  // the heads of the same tokens were fetched at other times. Neighbouring heads
  // of a unit are fetched together.
  static constexpr int kGroups = kWarps / HP;        // warps that share a head's tokens
  static constexpr int kTile = 16 * KT * kGroups;
  static constexpr int kHead = kTile * kHD * (kFp8 ? 1 : 2);  // bytes of a head's K (or V) tile
  static constexpr int kKV = HP * kHead;
  static constexpr int kStage = 2 * kKV;
  // CTAs an SM holds, and stages that fit its shared memory then
  static constexpr int kCtas = kFp8 && NT == 1 ? 3 : 2;
  static constexpr int kStages = kFp8 && (NT == 1 || HP == 2) ? 2 : 3;
  static constexpr int kScratch = kGroups > 1 ? HP * kRows * kScratchStride * 4 : 0;
  static constexpr int kSmem = kStages * kStage + kScratch + 1024;
};

// 16-byte chunk of a token's row in a tile: e4m3 rows are 128 bytes; bf16 rows
// two halves of 64 dims, a half tile apart. 128-byte swizzle.
template <bool kFp8>
__device__ __forceinline__ uint32_t swz(uint32_t base, int row, int chunk) {
  if constexpr (kFp8) return base + row * 128 + ((chunk ^ (row & 7)) << 4);
  return base + (chunk >> 3) * (64 * 128) + row * 128 + ((((chunk & 7) ^ (row & 7))) << 4);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// A load without the evict-first hint, for rows that are read again soon.
__device__ __forceinline__ void tma_load_4d_keep(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// Adds bytes to the transactions the barrier's current phase waits for.
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// four e4m3 bytes -> halves (exact)
__device__ __forceinline__ void e4m3x4_to_half(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Transpose of an 8x8 matrix of 16-bit values held one row per four lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
// Packed fp32 pairs.
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void un2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Bit i: row i of a warp's 16 KT rows of V, from row tok0 of the e4m3 tile at vb, holds a value that is not zero.
template <int KT>
__device__ __forceinline__ uint32_t rows_that_hold(uint32_t vb, int tok0, int lane) {
  uint32_t holds = 0;
#pragma unroll 1
  for (int i = 0; i < 4 * KT; ++i) {  // four rows at a time, eight lanes a row
    uint32_t x[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(swz<true>(vb, tok0 + i * 4 + (lane >> 3), lane & 7)));
    const uint32_t lanes = __ballot_sync(0xffffffffu, ((x[0] | x[1] | x[2] | x[3]) & 0x7f7f7f7fu) != 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) holds |= (uint32_t)((lanes >> (8 * r) & 0xffu) != 0) << (i * 4 + r);
  }
  return holds;
}

template <bool kFp8, int NT, int HP>
__global__ void __launch_bounds__(kThreads, (Cfg<kFp8, NT, HP>::kCtas))
    tree_warp_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ Args a) {
  using C = Cfg<kFp8, NT, HP>;
  static_assert(C::kCtas * (C::kSmem + 1408 + 1024) <= 228 * 1024, "the CTAs of an SM share its memory (with 1.4 KB of static, 1 KB reserved each)");
  constexpr int kRows = C::kRows, KT = C::KT, kTile = C::kTile;
  kernel_entry();
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::kStages];
  __shared__ __align__(8) uint64_t empty_bar[C::kStages];
  __shared__ __align__(16) uint8_t scales[C::kStages][2][HP * kTile];
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
        const int boxes = kTile / a.box;
        tree::Pages pg;
        pg.start(a, w, w.t0 * kTile);
        for (int j = 0; j < w.n; ++j, ++it) {
          const int s = it % C::kStages;
          if (it >= C::kStages && !mbar_wait(smem_u32(&empty_bar[s]), (it / C::kStages - 1) & 1, &g_err_tree)) {
            ok = false;
            break;
          }
          const uint32_t st = smem_u32(smem + s * C::kStage);
          const uint32_t fb = smem_u32(&full_bar[s]);
          // a tile is one box, or two when the pages hold 64 tokens (their second
          // half may lie past the sequence: it is read as zeros then)
          for (int x = 0; x < boxes; ++x) {
            const bool bad = pg.absent(a, w);
            const int blk = bad ? a.num_blocks : pg.blk;  // out of the tensor map: TMA fills zeros
            const int off = pg.off;
            if (kFp8 && bad) {  // a block outside the pool reads zeros, of scale 1
              for (int i = 0; i < 2; ++i)
                for (int h = 0; h < HP; ++h)
                  for (int k = 0; k < a.box / 4; ++k)
                    reinterpret_cast<uint32_t*>(&scales[s][i][h * kTile + x * a.box])[k] = 0x7f7f7f7fu;
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before a later copy into the same bytes
            }
            const uint32_t bytes = 2 * (C::kKV / boxes) + (kFp8 && !bad ? 2 * HP * a.box : 0);
            if (x + 1 < boxes)
              mbar_expect_tx(fb, bytes);
            else
              mbar_arrive_expect_tx(fb, bytes);
            for (int v = 0; v < 2; ++v)
#pragma unroll
              for (int h = 0; h < HP; ++h) {
                const uint32_t dst = st + v * C::kKV + h * C::kHead + x * a.box * 128;
                tma_load_4d(dst, v ? &vmap : &kmap, 0, w.h + h, off, blk, fb, pol);
                if constexpr (!kFp8) tma_load_4d(dst + C::kHead / 2, v ? &vmap : &kmap, 64, w.h + h, off, blk, fb, pol);
              }
            if (kFp8 && !bad) {
              const int64_t so = blk * a.scale_stride + (int64_t)w.h * a.block_size + off;
#pragma unroll
              for (int h = 0; h < HP; ++h) {
                bulk_load(smem_u32(&scales[s][0][h * kTile + x * a.box]), a.ks + so + (int64_t)h * a.block_size, a.box, fb);
                bulk_load(smem_u32(&scales[s][1][h * kTile + x * a.box]), a.vs + so + (int64_t)h * a.block_size, a.box, fb);
              }
            }
            pg.advance(a, w, a.box);
          }
        }
      }
      w.leave(a);
      // no copy may outlive the CTA: wait (bounded) for the last phase of every stage
      for (uint32_t i = it < C::kStages ? 0 : it - C::kStages; i < it; ++i)
        mbar_wait(smem_u32(&full_bar[i % C::kStages]), (i / C::kStages) & 1, &g_err_tree);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  // Lane (g, j4): tokens g and g + 8 of the warp's sixteen and query rows
  // 8 t + 2 j4, + 1 of S^T; the same rows and the dims of dim_of() of O^T.
  const int g = lane >> 2, j4 = lane & 3, mi = lane >> 3;
  const int hw = warp % HP, turn_of = warp / HP;  // this warp's head of the unit and place among its warps
  const int tok0 = turn_of * 16 * KT;
  // shared-memory offsets of this lane's rows in ldmatrix: 4 pairs of chunks;
  // chunks of a bf16 row's other half and the other tokens are constants apart
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    koff[i] = swz<kFp8>(0, tok0 + (lane & 7) + ((mi & 1) << 3), i * 2 + (mi >> 1));
    voff[i] = kFp8 ? koff[i] : swz<kFp8>(0, tok0 + (lane & 7) + ((mi >> 1) << 3), i * 2 + (mi & 1));
  }
  uint32_t it = 0;
  bool ok = true;
  while (w.next(a)) {
    const int base = w.s.len - w.s.nodes;  // position of node 0 (negative: earlier nodes are not in the cache)
    uint32_t qb[NT][8][2];
    float rscale[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // B fragments: this lane loads row 8 t + g
      const int R = w.rb * kRows + t * 8 + g, node = R / a.group;
      const bool in = node < w.s.nodes;
      const bf16* qp = a.q + (int64_t)(w.s.q0 + (in ? node : 0)) * a.q_st +
                       (int64_t)((w.h + hw) * a.group + (in ? R - node * a.group : 0)) * a.q_sh;
      if constexpr (kFp8) {
        // the row over a power of two as halves: exact to 2^-25 of its largest
        // finite value, which is brought to [1, 2); to less than 2^16 where that is
        // 2^113 or more, and to 2^-14 at least (the scale stays a normal number)
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
        const int e = min(max((int)(mx >> 7) - 127, -112), 112);
        const float inv = pow2(-e);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].x));
          const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].y));
          qb[t][ks][0] = pack_half(x.x * inv, x.y * inv);
          qb[t][ks][1] = pack_half(y.x * inv, y.y * inv);
        }
        const float mine = a.scale_log2 * pow2(e);
        rscale[t][0] = __shfl_sync(0xffffffffu, mine, j4 * 8);
        rscale[t][1] = __shfl_sync(0xffffffffu, mine, j4 * 8 + 4);
      } else {
        rscale[t][0] = rscale[t][1] = a.scale_log2;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          qb[t][ks][0] = in ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + j4 * 2) : 0u;
          qb[t][ks][1] = in ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + j4 * 2 + 8) : 0u;
        }
      }
    }
    float o[NT][8][4];
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int c = 0; c < 8; ++c) o[t][c][0] = o[t][c][1] = o[t][c][2] = o[t][c][3] = 0.f;
      m_run[t][0] = m_run[t][1] = -INFINITY;
      l_run[t][0] = l_run[t][1] = 0.f;
    }

    for (int jt = 0; jt < w.n && ok; ++jt, ++it) {
      const int s = it % C::kStages;
      if (!mbar_wait(smem_u32(&full_bar[s]), (it / C::kStages) & 1, &g_err_tree)) {
        ok = false;
        break;
      }
      const uint32_t kb = smem_u32(smem + s * C::kStage) + hw * C::kHead, vb = kb + C::kKV;
      const int p0 = (w.t0 + jt) * kTile + tok0;  // position of this warp's first token
      bool odd_v = false;                          // a node's V row holds a value that is not finite
      const bool tail = p0 + 16 * KT > base;
      if (tail) {
        // The warp's tokens reach into the draft or past the context. Rows past
        // the context hold stale bytes (possibly NaN): zero them, since a zero
        // weight does not cancel NaN. Drafted rows may be hidden from some of
        // the query rows: look for values that a zero weight would not cancel.
        for (int idx = lane; idx < 16 * KT * (kFp8 ? 8 : 16); idx += 32) {
          const int row = kFp8 ? idx >> 3 : idx >> 4, chunk = kFp8 ? idx & 7 : idx & 15;
          const uint32_t ad = swz<kFp8>(vb, tok0 + row, chunk);
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
        __syncwarp();  // the zeros are read by other lanes (a vote orders no memory)
      }

      // S^T of 16 tokens k: element 2 h + i is token 16 k + g + 8 h, row 8 t + 2 j4 + i
      float sc[KT][NT][4];
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[k][t][0] = sc[k][t][1] = sc[k][t][2] = sc[k][t][3] = 0.f;
      if constexpr (kFp8) {
        // k-step ks covers 16 dims; lane j4 holds dims 4 j4 .. 4 j4 + 3 of it,
        // for K and Q alike (any order of the dims gives the same sum)
#pragma unroll
        for (int kp = 0; kp < 4; ++kp)
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            uint32_t b[4];
            ldmatrix_x4(kb + koff[kp] + k * 2048, b[0], b[1], b[2], b[3]);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t ka[4];
              e4m3x4_to_half(b[2 * q], ka[0], ka[2]);
              e4m3x4_to_half(b[2 * q + 1], ka[1], ka[3]);
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_f16_16816(sc[k][t], ka, qb[t][kp * 2 + q][0], qb[t][kp * 2 + q][1]);
            }
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t ka[4];
          ldmatrix_x4(kb + koff[ks & 3] + (ks >> 2) * (64 * 128), ka[0], ka[1], ka[2], ka[3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_bf16_16816(sc[0][t], ka, qb[t][ks][0], qb[t][ks][1]);
        }
      }

      float ev[KT][2], vs[KT][2];  // exponents b and scales 2^b of the V rows of this lane's tokens
      bool unit = false;           // an exponent is 0
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (kFp8) {
            const int tk = hw * kTile + tok0 + k * 16 + g + 8 * h;
            const uint32_t kc = scales[s][0][tk], vc = scales[s][1][tk];
            const float ksc = __uint_as_float(kc << 23);
            ev[k][h] = __uint_as_float(0x4b000000u | vc) - (8388608.f + 127.f);  // vc - 127
            vs[k][h] = __uint_as_float(vc << 23);
            unit |= vc == 127u;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              float* x = &sc[k][t][2 * h];
              un2(mul2(pk2(x[0], x[1]), mul2(pk2(rscale[t][0], rscale[t][1]), pk2(ksc, ksc))), x[0], x[1]);
            }
          } else {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 2; ++i) sc[k][t][2 * h + i] *= rscale[t][i];
          }
        }
      if (kFp8 && __any_sync(0xffffffffu, unit)) {  // rare: rows of nothing, or with values between 224 and 448
        const uint32_t holds = rows_that_hold<KT>(vb, tok0, lane);
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (ev[k][h] == 0.f && !((holds >> (k * 16 + g + 8 * h)) & 1u)) ev[k][h] = kNothing, vs[k][h] = 0.f;
      }
      uint32_t hidden[KT];  // bit 4 t + 2 h + i: that score is masked
      if (tail) {
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          hidden[k] = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int pos = p0 + k * 16 + g + 8 * h;
            if (kFp8 && vs[k][h] == INFINITY) vs[k][h] = 0.f;  // stale scale bytes
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int node = (w.rb * kRows + t * 8 + 2 * j4 + i) / a.group;
                const bool seen = pos < base || (pos < w.s.len && node < w.s.nodes &&
                                                 tree::sees(a, w.s.q0 + node, node, pos - base));
                if (!seen) {
                  sc[k][t][2 * h + i] = -INFINITY;
                  hidden[k] |= 1u << (4 * t + 2 * h + i);
                }
              }
          }
        }
      }
      float half[NT][2];   // a row's references before this tile and after it: the root of the factor between them
      bool moved = false;  // a maximum of the warp's rows rose
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float mx[2] = {-INFINITY, -INFINITY}, ref[2];
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x0 = sc[k][t][2 * h], x1 = sc[k][t][2 * h + 1];
            if constexpr (kFp8) un2(add2(pk2(x0, x1), pk2(ev[k][h], ev[k][h])), x0, x1);
            mx[0] = fmaxf(mx[0], x0);
            mx[1] = fmaxf(mx[1], x1);
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 4));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 8));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 16));
          const float m_new = fmaxf(m_run[t][i], mx[i]);
          const float top = m_new == -INFINITY ? 0.f : m_new;
          ref[i] = kFp8 ? top - kTop : top;
          moved |= mx[i] > m_run[t][i];
          half[t][i] = ex2(0.5f * (m_run[t][i] - top));
          m_run[t][i] = m_new;
        }
        const uint64_t nref = pk2(-ref[0], -ref[1]);
        uint64_t sum = 0;
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float* x = &sc[k][t][2 * h];
            un2(add2(pk2(x[0], x[1]), nref), x[0], x[1]);
            x[0] = ex2(x[0]);
            x[1] = ex2(x[1]);
            const uint64_t w = pk2(x[0], x[1]);
            sum = add2(sum, w);
            if constexpr (kFp8) un2(mul2(w, pk2(vs[k][h], vs[k][h])), x[0], x[1]);
          }
        const uint64_t f = pk2(half[t][0], half[t][1]);
        un2(fma2(mul2(pk2(l_run[t][0], l_run[t][1]), f), f, sum), l_run[t][0], l_run[t][1]);
      }
      if (__any_sync(0xffffffffu, moved)) {  // rarely after a row's first tiles; otherwise every factor is 1
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][c][i] *= half[t][i & 1] * half[t][i & 1];
      }
      if (!odd_v) {
        // the weights are rounded to the type of the V operand: bf16 (2^-8 of each), or half (2^-11) for e4m3
        uint32_t pb[KT][NT][2];
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              pb[k][t][h] = transpose8(kFp8 ? pack_half(sc[k][t][2 * h], sc[k][t][2 * h + 1])
                                            : pack_bf16(sc[k][t][2 * h], sc[k][t][2 * h + 1]));
        if constexpr (kFp8) {
          // A transposed 8x8 of 16-bit elements gives a lane two tokens of a
          // pair of dims; a byte permutation pairs the tokens of each dim. Row
          // g of the MMA is dim 2 g of the 16-dim chunk, row g + 8 dim 2 g + 1.
#pragma unroll
          for (int cp = 0; cp < 4; ++cp)
#pragma unroll
            for (int k = 0; k < KT; ++k) {
              uint32_t b[4];
              ldmatrix_x4_trans(vb + voff[cp] + k * 2048, b[0], b[1], b[2], b[3]);
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                uint32_t va[4];
                e4m3x4_to_half(__byte_perm(b[2 * q], 0, 0x3120), va[0], va[1]);
                e4m3x4_to_half(__byte_perm(b[2 * q + 1], 0, 0x3120), va[2], va[3]);
#pragma unroll
                for (int t = 0; t < NT; ++t) mma_f16_16816(o[t][2 * cp + q], va, pb[k][t][0], pb[k][t][1]);
              }
            }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t va[4];
            ldmatrix_x4_trans(vb + voff[c & 3] + (c >> 2) * (64 * 128), va[0], va[1], va[2], va[3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_bf16_16816(o[t][c], va, pb[0][t][0], pb[0][t][1]);
          }
        }
      } else {
        // a drafted V row that is not finite: add only what each row sees, token
        // by token (rare, so it is written for size)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll 1
          for (int tk = 0; tk < 16; ++tk) {
            const int src = (tk & 7) * 4 + j4, h = tk >> 3, row = tok0 + 16 * k + tk;
            const uint32_t hid = __shfl_sync(0xffffffffu, hidden[k], src);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const float p0t = __shfl_sync(0xffffffffu, h ? sc[k][t][2] : sc[k][t][0], src);
              const float p1t = __shfl_sync(0xffffffffu, h ? sc[k][t][3] : sc[k][t][1], src);
              const bool see0 = !((hid >> (4 * t + 2 * h)) & 1u), see1 = !((hid >> (4 * t + 2 * h + 1)) & 1u);
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                float v0, v1;  // this lane's two dims of chunk c
                if constexpr (kFp8) {
                  uint32_t h01, unused;
                  e4m3x4_to_half(lds16(swz<kFp8>(vb, row, c) + g * 2), h01, unused);
                  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h01));
                  v0 = v.x, v1 = v.y;
                } else {
                  v0 = __uint_as_float(lds16(swz<kFp8>(vb, row, 2 * c) + g * 2) << 16);
                  v1 = __uint_as_float(lds16(swz<kFp8>(vb, row, 2 * c + 1) + g * 2) << 16);
                }
                if (see0) o[t][c][0] += p0t * v0, o[t][c][2] += p0t * v1;
                if (see1) o[t][c][1] += p1t * v0, o[t][c][3] += p1t * v1;
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

    // ------------------------------------------- join the warps of a head
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l_run[t][i] += __shfl_xor_sync(0xffffffffu, l_run[t][i], d);
    if constexpr (C::kGroups == 1) {
      // one warp holds the head: its fragments go straight to memory
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = t * 8 + 2 * j4 + i, R = w.rb * kRows + row, nd = R / a.group;
          const float M = ok ? m_run[t][i] : -INFINITY, L = ok ? l_run[t][i] : 0.f;
          if (nd >= w.s.nodes) continue;
          if (w.whole()) {
            const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing seen: 0
            bf16* op = a.out + (int64_t)(w.s.q0 + nd) * a.o_st + (int64_t)((w.h + hw) * a.group + R - nd * a.group) * a.o_sh;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint32_t*>(op + c * 16 + 2 * g) = pack_bf16(o[t][c][i] * inv, o[t][c][2 + i] * inv);
          } else {
            const int64_t pr = (((int64_t)blockIdx.x * 2 + w.slot()) * HP + hw) * kRows + row;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<float2*>(a.part_o + pr * kHD + c * 16 + 2 * g) = make_float2(o[t][c][i], o[t][c][2 + i]);
            if (g == 0) {
              a.part_m[pr] = M;
              a.part_l[pr] = L;
            }
          }
        }
    } else {
      if (g == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mw[warp][t * 8 + 2 * j4 + i] = m_run[t][i];
            lw[warp][t * 8 + 2 * j4 + i] = l_run[t][i];
          }
      }
      named_bar_sync(1, kWarps * 32);
      float f[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float M = -INFINITY;
#pragma unroll
          for (int v = 0; v < C::kGroups; ++v) M = fmaxf(M, mw[v * HP + hw][t * 8 + 2 * j4 + i]);
          // a warp whose tokens were all masked contributes nothing (its rows are 0)
          f[t][i] = m_run[t][i] == -INFINITY ? 0.f : ex2(m_run[t][i] - M);  // 0 far below M, as the rows are
        }
#pragma unroll 1
      for (int turn = 0; turn < C::kGroups; ++turn) {
        if (turn_of == turn) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float* at = scratch + (hw * kRows + t * 8 + 2 * j4 + i) * kScratchStride + c * 16;
                const float v0 = o[t][c][i] * f[t][i], v1 = o[t][c][2 + i] * f[t][i];
                if constexpr (kFp8) {
                  float2* p2 = reinterpret_cast<float2*>(at + 2 * g);
                  const float2 old = turn > 0 ? *p2 : make_float2(0.f, 0.f);
                  *p2 = make_float2(old.x + v0, old.y + v1);
                } else {
                  at[g] = (turn > 0 ? at[g] : 0.f) + v0;
                  at[8 + g] = (turn > 0 ? at[8 + g] : 0.f) + v1;
                }
              }
        }
        named_bar_sync(1, kWarps * 32);
      }
      constexpr int kDims = HP * kRows;  // dims of a thread: 128 threads share HP x kRows x 128 values
      const int hrow = threadIdx.x / (kHD / kDims), d0 = threadIdx.x % (kHD / kDims) * kDims;
      const int hh = hrow / kRows, row = hrow - hh * kRows;
      const int R = w.rb * kRows + row;
      const int nd = R / a.group;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int v = 0; v < C::kGroups; ++v) M = fmaxf(M, mw[v * HP + hh][row]);
#pragma unroll
      for (int v = 0; v < C::kGroups; ++v) {
        const float e = mw[v * HP + hh][row] == -INFINITY ? 0.f : ex2(0.5f * (mw[v * HP + hh][row] - M));
        L += lw[v * HP + hh][row] * e * e;  // keeps NaN
      }
      if (!ok) M = -INFINITY, L = 0.f;
      const float* sp = scratch + hrow * kScratchStride + d0;
      if (nd < w.s.nodes) {
        if (w.whole()) {
          const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing seen: 0
          bf16* op =
              a.out + (int64_t)(w.s.q0 + nd) * a.o_st + (int64_t)((w.h + hh) * a.group + R - nd * a.group) * a.o_sh + d0;
#pragma unroll
          for (int c = 0; c < kDims / 8; ++c) {
            uint4 y;
            y.x = pack_bf16(sp[8 * c] * inv, sp[8 * c + 1] * inv);
            y.y = pack_bf16(sp[8 * c + 2] * inv, sp[8 * c + 3] * inv);
            y.z = pack_bf16(sp[8 * c + 4] * inv, sp[8 * c + 5] * inv);
            y.w = pack_bf16(sp[8 * c + 6] * inv, sp[8 * c + 7] * inv);
            reinterpret_cast<uint4*>(op)[c] = y;
          }
        } else {
          const int64_t pr = (((int64_t)blockIdx.x * 2 + w.slot()) * HP + hh) * kRows + row;
          float4* dst = reinterpret_cast<float4*>(a.part_o + pr * kHD + d0);
#pragma unroll
          for (int c = 0; c < kDims / 4; ++c) dst[c] = make_float4(sp[4 * c], sp[4 * c + 1], sp[4 * c + 2], sp[4 * c + 3]);
          if (d0 == 0) {
            a.part_m[pr] = M;
            a.part_l[pr] = L;
          }
        }
      }
      named_bar_sync(1, kWarps * 32);  // scratch and statistics are free again
    }
  }
}

}  // namespace
}  // namespace kvb

#include "tree_attn_tc.cuh"

namespace kvb {
namespace {

// ------------------------------------------------------------------- merge
// Joins the pieces of units that were cut between CTAs, in an order that does
// not depend on timing, and writes zeros for sequences with an empty context.
// Rows whose unit was whole have been written already.
constexpr int kMergeWarps = 8;
constexpr int kMergeCtas = 5;  // blocks an SM holds
constexpr int kFew = 16;

struct Joined {
  float m, l;
  float4 o;
};
__device__ __forceinline__ void join(Joined& x, float m, float l, const float4& o) {
  const float m_new = fmaxf(x.m, m);
  // A part in which the row saw nothing (m = -inf) adds 0. The sums are scaled in two
  // steps: they count even where the rows, far below the new reference, do not.
  const float h0 = x.m == -INFINITY ? 0.f : ex2(0.5f * (x.m - m_new)), h1 = m == -INFINITY ? 0.f : ex2(0.5f * (m - m_new));
  const float f0 = h0 * h0, f1 = h1 * h1;
  x.l = x.l * h0 * h0 + l * h1 * h1;
  x.o.x = x.o.x * f0 + o.x * f1;
  x.o.y = x.o.y * f0 + o.y * f1;
  x.o.z = x.o.z * f0 + o.z * f1;
  x.o.w = x.o.w * f0 + o.w * f1;
  x.m = m_new;
}
// Pieces k0, k0 + step, .. < n of four dims of a row, from part p on; loads of four in flight.
__device__ __forceinline__ Joined join_parts(const Args& a, int p, int n, int k0, int step, int row, int chunk) {
  Joined x = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int k = k0; k < n; k += 4 * step) {
    float m[4], l[4];
    float4 o[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int kk = k + u * step;
      m[u] = -INFINITY;
      l[u] = 0.f;
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (kk < n) {
        // the unit's first part holds its beginning (slot 1), the others follow on (slot 0)
        const int64_t first = ((int64_t)(p + kk) * 2 + (kk == 0)) * a.heads * a.rows, pr = first + row;
        m[u] = a.part_m[pr];
        l[u] = a.part_l[pr];
        o[u] = reinterpret_cast<const float4*>(a.part_o)[a.by_dims ? first * 32 + (int64_t)chunk * a.rows + row : pr * 32 + chunk];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) join(x, m[u], l[u], o[u]);
  }
  return x;
}

// Only the cut units are looked at, at most one a part: a block has some parts
// (blockIdx.x, at most 32) and takes eight rows of each unit (blockIdx.y), or, when
// it has many pieces, its warps share a warp's part of those rows (a row's four
// dims a thread). A warp for every query row of the batch,
// finding its pieces from prefix sums, took 40 us for 64 x 1024 rows of which a
// fifth was cut; this takes 12.
__global__ void __launch_bounds__(kMergeWarps * 32, kMergeCtas) tree_merge_kernel(const __grid_constant__ Args a) {
  kernel_entry();
  __shared__ Joined s_join[kMergeWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mine = blockIdx.x + lane * gridDim.x;
  uint32_t cut = __ballot_sync(0xffffffffu, mine < a.parts && a.cuts[mine].n != 0);
  for (; cut; cut &= cut - 1) {
    const int part = blockIdx.x + (__ffs(cut) - 1) * gridDim.x;
    const tree::Cut c = a.cuts[part];
    const bool many = c.n > kFew;
    const int items = ((a.heads * c.rows + 7) >> 3) * (many ? 8 : 1);
    for (int item = blockIdx.y; item < items; item += gridDim.y) {
      const int group = many ? item >> 3 : item, eighth = many ? item & 7 : warp;
      const int f = group * 8 + (a.by_dims ? lane & 7 : eighth);  // row of the unit, its heads one after another
      const int head = f / c.rows, r = f - head * c.rows;
      const int chunk = a.by_dims ? eighth * 4 + (lane >> 3) : lane;
      const int n = head < a.heads ? c.n : 0;
      Joined x = join_parts(a, part, n, many ? warp : 0, many ? kMergeWarps : 1, head * a.rows + r, chunk);
      if (many) {
        s_join[warp][lane] = x;
        __syncthreads();
      }
      if (many && warp == 0)
        for (int w = 1; w < kMergeWarps; ++w) join(x, s_join[w][lane].m, s_join[w][lane].l, s_join[w][lane].o);
      if (n > 0 && (!many || warp == 0)) {
        const float inv = x.l == 0.f ? 0.f : 1.f / x.l;
        const int R = c.row0 + r, nd = R / a.group;
        *reinterpret_cast<uint2*>(a.out + (int64_t)(c.q0 + nd) * a.o_st +
                                  (int64_t)((c.h + head) * a.group + R - nd * a.group) * a.o_sh + chunk * 4) =
            make_uint2(pack_bf16(x.o.x * inv, x.o.y * inv), pack_bf16(x.o.z * inv, x.o.w * inv));
      }
      if (many) __syncthreads();  // before the next item's s_join
    }
  }
  for (int b = blockIdx.y * gridDim.x + blockIdx.x; b < a.batch; b += gridDim.x * gridDim.y) {
    const tree::Seq s = tree::seq_of(a, b, false);
    if (s.tiles) continue;
    const int64_t chunks = (int64_t)s.nodes * a.hq * 32;
    for (int64_t i = threadIdx.x; i < chunks; i += kMergeWarps * 32) {
      const int row = (int)(i >> 5), nd = row / a.hq;
      *reinterpret_cast<uint2*>(a.out + (int64_t)(s.q0 + nd) * a.o_st + (int64_t)(row - nd * a.hq) * a.o_sh + (i & 31) * 4) =
          make_uint2(0u, 0u);
    }
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
                   CU_TENSOR_MAP_SWIZZLE_128B,
                   // an e4m3 row of one head is 128 bytes: a wider fetch would bring the next head's
                   fp8 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(kEncode, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
  return kOk;
}

// The kernel variant of a call, and what its launch needs.
struct Variant {
  int nt;  // eights of query rows a unit holds for the warp-MMA kernel; 0: the tcgen05 kernel
  int rows, heads, tile, box, parts;
  size_t workspace;
};

template <bool kFp8, int NT, int HP>
void fill(Variant* v) {
  using C = Cfg<kFp8, NT, HP>;
  v->nt = NT;
  v->rows = C::kRows;
  v->heads = HP;
  v->tile = C::kTile;
  v->parts = C::kCtas * device_sm_count();  // what the SMs hold: one wave
}

// More than 16 query rows a kv head over bf16 (8, while every sequence and kv head
// can have an SM), or 32 over e4m3 (two units of the warp-MMA kernel), take tcgen05.
// Warp MMAs against tcgen05, us:
// bf16, 256 sequences of 1024 tokens: 4 rows 169 / 211, 12 rows 186 / 214; 16 of
// 3900..8100: 8 rows 73 / 74, 16 rows 80 / 75, 32 rows 123 / 77; 16 rows over 8 heads: one
// of 100 16.4 / 14.4, 1531 19.5 / 18.5, 8000 21.5 / 22.8, 100000 81 / 78, 18 of 100..9000
// 84 / 66; above the SM count 32 of 500..1500 42 / 44, 128 of those 115 / 140, 32 of
// 3900..8100 137 / 135, 24 of 9000 152 / 148, but 20 of 100..9000 87 / 72 and 40 of
// 200..12000 183 / 167: only long and very uneven contexts lose there by the rule, and
// the host knows no lengths.
// e4m3, 256 of 1024: 16 rows 139 / 345, 32 rows 253 / 352; 16 of 3900..8100: 16 rows 58 /
// 97, 32 rows 92 / 99, 48 rows 129 / 103; 130001 tokens: 32 rows 41 / 43, 48 rows 50 / 45.
Variant variant_for(bool fp8, int batch, int hq, int hkv, int max_nodes, int block_size) {
  Variant v;
  const int64_t rows = (int64_t)(hq / hkv) * max_nodes;
  const bool few = rows <= 8;
  const int hp = !fp8 ? 1 : hkv % 4 == 0 ? 4 : hkv % 2 == 0 ? 2 : 1;
  const int most = fp8 ? 32 : (int64_t)batch * hkv <= device_sm_count() ? 8 : 16;  // rows for warp MMAs
  if (rows > most) {
    v.nt = 0;
    v.rows = tcore::kRows;
    v.heads = 1;
    v.tile = tcore::kTile;
    v.parts = device_sm_count();
  } else if (!fp8)
    few ? fill<false, 1, 1>(&v) : fill<false, 2, 1>(&v);
  else if (hp == 4)
    few ? fill<true, 1, 4>(&v) : fill<true, 2, 4>(&v);
  else if (hp == 2)
    few ? fill<true, 1, 2>(&v) : fill<true, 2, 2>(&v);
  else
    few ? fill<true, 1, 1>(&v) : fill<true, 2, 1>(&v);
  v.box = block_size % v.tile == 0 ? v.tile : 64;
  v.workspace = (size_t)v.parts * 2 * v.heads * v.rows * (kHD + 2) * sizeof(float) + (size_t)v.parts * sizeof(tree::Cut);
  return v;
}

template <bool kFp8>
int launch_tc(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  constexpr int kSmem = tcore::Cfg<kFp8>::kSmem;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "kvb_tree_attn: cudaGetDevice");
  if (dev >= 64 || !((done.load() >> dev) & 1ull)) {
    e = cudaFuncSetAttribute(tcore::tree_tc_kernel<kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return cuda_status(e, "kvb_tree_attn: shared memory attribute");
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  e = launch_kernel(tcore::tree_tc_kernel<kFp8>, dim3(a.parts), dim3(tcore::kThreads), kSmem, st, km, vm, a);
  return cuda_status(e, "kvb_tree_attn launch");
}

template <bool kFp8, int NT, int HP>
int launch_warp(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  constexpr int kSmem = Cfg<kFp8, NT, HP>::kSmem;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "kvb_tree_attn: cudaGetDevice");
  if (dev >= 64 || !((done.load() >> dev) & 1ull)) {
    e = cudaFuncSetAttribute(tree_warp_kernel<kFp8, NT, HP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return cuda_status(e, "kvb_tree_attn: shared memory attribute");
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  e = launch_kernel(tree_warp_kernel<kFp8, NT, HP>, dim3(a.parts), dim3(kThreads), kSmem, st, km, vm, a);
  return cuda_status(e, "kvb_tree_attn launch");
}

}  // namespace
}  // namespace kvb

using namespace kvb;

extern "C" int kvb_tree_attn_workspace_size(int batch, int num_q_heads, int num_kv_heads, int max_seqlen_q,
                                            size_t* bytes) {
  if (!bytes) return set_error(kInvalid, "kvb_tree_attn_workspace_size: bytes is NULL");
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || max_seqlen_q < 0)
    return set_error(kInvalid, "kvb_tree_attn_workspace_size: bad sizes");
  // the larger of the two cache types' needs (the block size does not matter)
  const size_t a = variant_for(false, batch, num_q_heads, num_kv_heads, max_seqlen_q, 256).workspace;
  const size_t b = variant_for(true, batch, num_q_heads, num_kv_heads, max_seqlen_q, 256).workspace;
  *bytes = a > b ? a : b;
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
  if (total_q * num_q_heads > INT32_MAX) return set_error(kUnsupported, "kvb_tree_attn: more than 2^31 query rows");
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
  const Variant v = variant_for(fp8, batch, num_q_heads, num_kv_heads, max_seqlen_q, block_size);
  a.rows = v.rows;
  a.by_dims = v.nt == 0;
  a.heads = v.heads;
  a.head_groups = num_kv_heads / v.heads;
  while ((1 << a.row_shift) < v.rows) ++a.row_shift;
  while ((1 << a.tile_shift) < v.tile) ++a.tile_shift;
  a.tile = v.tile;
  a.box = v.box;
  a.parts = v.parts;
  const size_t need = v.workspace;
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
  a.cuts = (tree::Cut*)workspace;
  a.part_o = (float*)(a.cuts + a.parts);
  a.part_m = a.part_o + (size_t)a.parts * 2 * a.heads * a.rows * kHD;
  a.part_l = a.part_m + (size_t)a.parts * 2 * a.heads * a.rows;
  a.scale_log2 = scale * 1.4426950408889634f;

  CUtensorMap km, vm;
  const int64_t bytes = block_stride * (fp8 ? 1 : 2);
  int rc = encode_pages(&km, k_cache, fp8, num_blocks, bytes, block_size, num_kv_heads, a.box);
  if (!rc) rc = encode_pages(&vm, v_cache, fp8, num_blocks, bytes, block_size, num_kv_heads, a.box);
  const cudaStream_t st = (cudaStream_t)stream;
  if (rc) return rc;
  if (v.nt == 0)
    rc = fp8 ? launch_tc<true>(km, vm, a, st) : launch_tc<false>(km, vm, a, st);
  else if (!fp8)
    rc = v.nt == 1 ? launch_warp<false, 1, 1>(km, vm, a, st) : launch_warp<false, 2, 1>(km, vm, a, st);
  else if (v.heads == 4)
    rc = v.nt == 1 ? launch_warp<true, 1, 4>(km, vm, a, st) : launch_warp<true, 2, 4>(km, vm, a, st);
  else if (v.heads == 2)
    rc = v.nt == 1 ? launch_warp<true, 1, 2>(km, vm, a, st) : launch_warp<true, 2, 2>(km, vm, a, st);
  else
    rc = v.nt == 1 ? launch_warp<true, 1, 1>(km, vm, a, st) : launch_warp<true, 2, 1>(km, vm, a, st);
  if (rc) return rc;
  // a block for each eight rows of a part's cut unit; where units are few and so cut in many pieces, a block for
  // each eighth of that and fewer parts a block, to have one wave
  const int64_t unit_rows = (int64_t)a.group * max_seqlen_q, blocks = (unit_rows + v.rows - 1) / v.rows;
  const int64_t units = (int64_t)batch * (num_kv_heads / v.heads) * blocks;
  const int eights = (int)((v.heads * (unit_rows < v.rows ? unit_rows : v.rows) + 7) / 8);
  const bool few = units * kFew <= v.parts;
  const int y = few ? eights * 8 : eights;
  const int wave = kMergeCtas * device_sm_count() / y, least = (v.parts + 31) / 32;
  const int x = !few || wave >= v.parts ? v.parts : wave > least ? wave : least;
  return cuda_status(launch_kernel(tree_merge_kernel, dim3((unsigned)x, (unsigned)y), dim3(kMergeWarps * 32), 0, st, a),
                     "kvb_tree_attn merge launch");
}
