// The tensor-core form of the tree attention, for units of more than 16 query
// rows: included by tree_attn.cu.
//
// A CTA owns 128 query rows (nodes x query heads of one kv head) and walks the
// context in 128-token tiles: S = Q K^T is a tcgen05.mma chain into TMEM, two
// softmax warpgroups take the tiles in turn (one thread per query row, so no
// reduction crosses threads), write the weights P to shared memory and fold
// P V, a second tcgen05.mma chain, into their own fp32 rows. The two groups keep
// separate maxima and sums, which are joined at the end of a segment, so one
// group's exponentials overlap the other group's MMAs. One warp issues the TMA
// loads, one thread the MMAs.
//
// Over an e4m3 cache the operands stay e4m3: Q and P are split in two e4m3 parts,
// x = hi + lo, hi = e4m3(x), lo = e4m3(x - hi). Two 4-bit significands with the
// lower one signed hold a bf16 query exactly (its 8 bits) down to 2^-10 of the
// row's maximum, scaled to [128, 256), and 2^-18 of that maximum below it; a weight
// scaled by 2^8 likewise, so its error is at most 2^-9 of itself or 2^-18 of the
// row's largest. Two e4m3 chains take as long as one bf16 chain, K and V are never
// converted, and their tiles are half as large.
#pragma once

namespace kvb {
namespace {
namespace tcore {

constexpr int kRows = 128;
constexpr int kTile = 128;
constexpr int kGroups = 2;                                // softmax warpgroups
constexpr int kThreads = 128 + kGroups * 128;             // warp 0 TMA, warp 1 MMA + TMEM, warps 2 and 3 idle
// Registers: 168 a thread at launch (384 threads); the control warps give theirs
// up for the softmax threads' output rows: 128 (56 + 2 * 224) = 384 * 168.
constexpr int kControlRegs = 56, kSoftmaxRegs = 224;
constexpr uint32_t kCols = 512;                           // S0, S1, PV0, PV1 (128 columns each)
constexpr int kOperand = kRows * kHD * 2;                 // Q or P: bf16, or two e4m3 parts
constexpr int kPart = kOperand / 2;                       // an e4m3 part, or 64 columns of bf16
template <bool kFp8>
struct Cfg {
  static constexpr int kKV = kTile * kHD * (kFp8 ? 1 : 2);
  static constexpr int kStage = 2 * kKV;
  static constexpr int kStages = kFp8 ? 3 : 2;
  static constexpr int kQ = 0, kP = kOperand, kRing = (1 + kGroups) * kOperand;
  static constexpr int kSmem = kRing + kStages * kStage + 1024;
};
// K-major operand rows of 128 bytes, 128-byte swizzle: 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// V as the B operand of P V (head dim contiguous): 128-byte atoms along the head
// dim `apart` bytes apart (bf16: two halves; e4m3: one atom holds all 128 dims),
// 8-token groups 1024 B apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t apart) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(apart >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <bool kFp8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (kFp8)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ bool any_of_barrier(int id, int threads, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  return __uint_as_float(r);
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four values as hi and lo e4m3 parts.
__device__ __forceinline__ void split4(const float* x, uint32_t& hi, uint32_t& lo) {
  const uint32_t h01 = to_e4m3x2(x[0], x[1]), h23 = to_e4m3x2(x[2], x[3]);
  hi = h01 | h23 << 16;
  uint32_t a, b;
  e4m3x4_to_half(hi, a, b);
  const float2 f01 = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 f23 = __half22float2(*reinterpret_cast<const __half2*>(&b));
  lo = to_e4m3x2(x[0] - f01.x, x[1] - f01.y) | to_e4m3x2(x[2] - f23.x, x[3] - f23.y) << 16;
}

// Bits of the 32 tokens from position pos0 that a row sees (a row: node i, mask row `row`).
__device__ __forceinline__ uint32_t seen32(const Args& a, int row, int i, int base, int len, int pos0) {
  const int k = len - pos0;
  uint32_t m = k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
  const int rel = pos0 - base;  // node index of the first token
  if (rel + 32 > 0 && m) {
    uint32_t t;
    if (!a.mask) {
      const int n = i - rel + 1;
      t = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
    } else {
      const uint32_t* w = a.mask + (int64_t)row * a.mask_stride;
      if (rel >= 0) {
        const int w0 = rel >> 5;
        const uint32_t lo = w0 < a.mask_words ? w[w0] : 0u, hi = w0 + 1 < a.mask_words ? w[w0 + 1] : 0u;
        t = __funnelshift_r(lo, hi, rel & 31);
      } else {
        t = w[0] << -rel | ((1u << -rel) - 1u);
      }
    }
    m &= t;
  }
  return m;
}

template <bool kFp8>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ Args a) {
  using C = Cfg<kFp8>;
  kernel_entry();
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full, kfull[C::kStages], vfull[C::kStages], kv_empty[C::kStages], s_full[2], s_empty[2],
      p_full[2], pv_full[2], pv_empty[2];
  __shared__ __align__(16) uint8_t scales[kFp8 ? C::kStages : 1][2][kTile];
  // a tile's scales 2^a (K) and 2^b (V) as floats: 2^a, b and 2^-b
  __shared__ __align__(16) float tok_k[kFp8 ? 2 : 1][kTile], tok_b[kFp8 ? 2 : 1][kTile], tok_i[kFp8 ? 2 : 1][kTile];
  __shared__ float m_other[kRows], l_other[kRows];
  __shared__ uint32_t odd_bits[2][4];
  __shared__ uint32_t tmem_s;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&q_full), kGroups * 4);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(smem_u32(&kfull[i]), 1);
      mbar_init(smem_u32(&vfull[i]), 1);
      mbar_init(smem_u32(&kv_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&s_empty[i]), 4);
      mbar_init(smem_u32(&p_full[i]), 4);
      mbar_init(smem_u32(&pv_full[i]), 1);
      mbar_init(smem_u32(&pv_empty[i]), 4);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::fence_before();
  const tree::Start start = tree::find_start<kThreads>(a, blockIdx.x);  // synchronises the block
  tc::fence_after();
  const uint32_t tmem = tmem_s;
  Walk w(a, start);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
    if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
      const uint64_t pol = l2_evict_first_policy();
      uint32_t it = 0;
      bool ok = true;
      while (ok && w.next(a)) {
        // several row blocks read the same rows: keep those in L2
        const bool once = w.s.blocks == 1;
        int col = -1, blk = 0;
        bool bad = false;
        for (int j = 0; j < w.n; ++j, ++it) {
          const int st = it % C::kStages;
          if (it >= C::kStages && !mbar_wait(smem_u32(&kv_empty[st]), (it / C::kStages - 1) & 1, &g_err_tree)) {
            ok = false;
            break;
          }
          const int t0 = (w.t0 + j) * kTile;
          const uint32_t kd = sbase + C::kRing + st * C::kStage, vd = kd + C::kKV;
          const uint32_t kb = smem_u32(&kfull[st]), vb = smem_u32(&vfull[st]);
          const int boxes = kTile / a.box;
          for (int x = 0; x < boxes; ++x) {
            const int at = t0 + x * a.box;
            if (at / a.block_size != col) {
              col = at / a.block_size;
              const bool past = at >= w.s.len;
              blk = past ? -1 : a.tables[(int64_t)w.b * a.bt_stride + col];
              bad = blk < 0 || blk >= a.num_blocks;
              if (bad) {
                if (!past) atomicOr(&g_err_tree, (unsigned)kErrBlockTable);
                blk = a.num_blocks;  // out of the tensor map: TMA fills zeros
              }
            }
            const int off = at - col * a.block_size;
            if (kFp8 && bad) {  // a block outside the pool reads zeros, of scale 1
              for (int i = 0; i < 2; ++i)
                for (int k = 0; k < a.box / 4; ++k)
                  reinterpret_cast<uint32_t*>(&scales[st][i][x * a.box])[k] = 0x7f7f7f7fu;
              fence_async();  // before a later copy into the same bytes
            }
            const uint32_t bytes = C::kKV / boxes;
            const uint32_t more = kFp8 && !bad ? 2 * a.box : 0;  // the scales come with K
            if (x + 1 < boxes) {
              mbar_expect_tx(kb, bytes + more);
              mbar_expect_tx(vb, bytes);
            } else {
              mbar_arrive_expect_tx(kb, bytes + more);
              mbar_arrive_expect_tx(vb, bytes);
            }
            if (kFp8 && !bad) {
              const int64_t so = blk * a.scale_stride + (int64_t)w.h * a.block_size + off;
              bulk_load(smem_u32(&scales[st][0][x * a.box]), a.ks + so, a.box, kb);
              bulk_load(smem_u32(&scales[st][1][x * a.box]), a.vs + so, a.box, kb);
            }
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
              for (int hf = 0; hf < (kFp8 ? 1 : 2); ++hf) {
                const uint32_t dst = (v ? vd : kd) + hf * kPart + x * a.box * 128;
                if (once)
                  tma_load_4d(dst, v ? &vmap : &kmap, hf * 64, w.h, off, blk, v ? vb : kb, pol);
                else
                  tma_load_4d_keep(dst, v ? &vmap : &kmap, hf * 64, w.h, off, blk, v ? vb : kb);
              }
          }
        }
      }
      // no copy may outlive the CTA: wait (bounded) for the last phase of every stage
      for (uint32_t i = it < C::kStages ? 0 : it - C::kStages; i < it; ++i) {
        mbar_wait(smem_u32(&kfull[i % C::kStages]), (i / C::kStages) & 1, &g_err_tree);
        mbar_wait(smem_u32(&vfull[i % C::kStages]), (i / C::kStages) & 1, &g_err_tree);
      }
    }
    } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      // fp32 accumulation, M = N = 128, bf16 or e4m3 operands; V is read head-dim-major (bit 16)
      constexpr uint32_t kIdesc = (1u << 4) | (kFp8 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(kTile >> 3) << 17) |
                                  ((uint32_t)(kRows >> 4) << 24);
      constexpr int kParts = kFp8 ? 2 : 1, kSteps = kFp8 ? 4 : 8;  // MMAs of 32 or 16 along K
      uint32_t it = 0, seg = 0, done[2] = {0, 0};                  // tiles, segments, tiles of each group so far
      bool ok = true;
      while (ok && w.next(a)) {
        if (!mbar_wait(smem_u32(&q_full), seg & 1, &g_err_tree)) break;
        ++seg;
        const auto issue_s = [&](int j) -> bool {
          const int gr = j & 1;
          const uint32_t i = it + j, st = i % C::kStages, use = done[gr] + (j >> 1);
          if (use >= 1 && !mbar_wait(smem_u32(&s_empty[gr]), (use - 1) & 1, &g_err_tree)) return false;
          if (!mbar_wait(smem_u32(&kfull[st]), (i / C::kStages) & 1, &g_err_tree)) return false;
          tc::fence_after();
          const uint32_t q = sbase + C::kQ, k = sbase + C::kRing + st * C::kStage;
#pragma unroll
          for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
              const uint32_t off = (kFp8 ? 0 : (ks >> 2) * kPart) + (ks & 3) * 32;
              mma<kFp8>(tmem + gr * 128, desc_k(q + part * kPart + off), desc_k(k + off), kIdesc, part > 0 || ks > 0);
            }
          commit(smem_u32(&s_full[gr]));
          return true;
        };
        ok = issue_s(0);
        for (int j = 0; j < w.n && ok; ++j) {
          if (j + 1 < w.n && !issue_s(j + 1)) {
            ok = false;
            break;
          }
          const int gr = j & 1;
          const uint32_t i = it + j, st = i % C::kStages, use = done[gr] + (j >> 1);
          ok = mbar_wait(smem_u32(&p_full[gr]), use & 1, &g_err_tree) &&
               mbar_wait(smem_u32(&vfull[st]), (i / C::kStages) & 1, &g_err_tree) &&
               (use == 0 || mbar_wait(smem_u32(&pv_empty[gr]), (use - 1) & 1, &g_err_tree));
          if (!ok) break;
          tc::fence_after();
          const uint32_t p = sbase + C::kP + gr * kOperand, v = sbase + C::kRing + st * C::kStage + C::kKV;
#pragma unroll
          for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
              const uint32_t off = (kFp8 ? 0 : (ks >> 2) * kPart) + (ks & 3) * 32;
              mma<kFp8>(tmem + (2 + gr) * 128, desc_k(p + part * kPart + off), desc_mn(v + ks * (kFp8 ? 4096 : 2048), kPart),
                        kIdesc | (1u << 16), part > 0 || ks > 0);
            }
          commit(smem_u32(&pv_full[gr]));
          commit(smem_u32(&kv_empty[st]));
        }
        it += w.n;
        done[0] += (w.n + 1) >> 1;
        done[1] += w.n >> 1;
      }
    }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------ softmax groups
    // A wait that gave up (its error bit is set) is not followed by others, and the
    // group goes on with what is there: its barriers stay matched, its rows are dropped.
    const int gr = (warp - 4) >> 2;                  // group: tiles of its parity
    const int qd = warp & 3;                         // TMEM lane quarter of this warp
    const int r = qd * 32 + lane;                    // query row of the unit = TMEM lane; token of a tile
    const int bar = 1 + gr;                          // the group's named barrier
    const uint32_t lane_base = tmem + ((uint32_t)(qd * 32) << 16);
    const uint32_t srow = lane_base + gr * 128, pvrow = lane_base + (2 + gr) * 128;
    const uint32_t pbase = sbase + C::kP + gr * kOperand;
    uint32_t it = 0, use = 0;
    bool ok = true;
    while (w.next(a)) {
      const int base = w.s.len - w.s.nodes;
      const int R = w.rb * kRows + r, node = R / a.group;
      const bool in = node < w.s.nodes;
      const int qrow = w.s.q0 + (in ? node : 0);
      const int head = w.h * a.group + (in ? R - node * a.group : 0);
      // -------- this thread's query row to shared memory: its half of the dims
      float rscale = a.scale_log2;
      {
        const uint4* qp = reinterpret_cast<const uint4*>(a.q + (int64_t)qrow * a.q_st + (int64_t)head * a.q_sh);
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (kFp8) {
          uint32_t mx = 0;
          bool finite = true;
#pragma unroll 4
          for (int c = 0; c < 16; ++c) {
            const uint4 x = in ? qp[c] : zero;
            const uint32_t wd[4] = {x.x & 0x7fff7fffu, x.y & 0x7fff7fffu, x.z & 0x7fff7fffu, x.w & 0x7fff7fffu};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t inf = __vcmpgtu2(wd[i], 0x7f7f7f7fu);
              finite &= inf == 0;
              mx = __vmaxu2(mx, wd[i] & ~inf);
            }
          }
          mx = max(mx & 0xffffu, mx >> 16);
          const int e = min(max((int)(mx >> 7) - 127 - 7, -100), 100);  // the largest to [128, 256)
          const float inv = pow2(-e);
          rscale = finite ? a.scale_log2 * pow2(e) : NAN;  // a row with NaN or an infinity gives NaN
#pragma unroll 1
          for (int c = gr * 8; c < gr * 8 + 8; c += 2) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint4 x = in ? qp[c + y] : zero;
              const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x);
              float f[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 v = __bfloat1622float2(h[i]);
                f[2 * i] = v.x * inv;
                f[2 * i + 1] = v.y * inv;
              }
              split4(f, hi[2 * y], lo[2 * y]);
              split4(f + 4, hi[2 * y + 1], lo[2 * y + 1]);
            }
            const uint32_t at = sbase + C::kQ + r * 128 + (((c >> 1) ^ (r & 7)) << 4);
            sts128(at, hi[0], hi[1], hi[2], hi[3]);
            sts128(at + kPart, lo[0], lo[1], lo[2], lo[3]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint4 x = in ? qp[gr * 8 + c] : zero;
            sts128(sbase + C::kQ + gr * kPart + r * 128 + ((c ^ (r & 7)) << 4), x.x, x.y, x.z, x.w);
          }
        }
      }
      fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&q_full));

      float o[kHD];
#pragma unroll
      for (int i = 0; i < kHD; ++i) o[i] = 0.f;
      float m_run = -INFINITY, l_run = 0.f;
      float corr_prev = 1.f;  // factor of the tile whose P V is folded next
      bool pending = false;
      // O = O * corr + P V of this group's last tile
      const auto fold = [&](float corr) {
        ok = ok && mbar_wait(smem_u32(&pv_full[gr]), (use - 1) & 1, &g_err_tree);
        tc::fence_after();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tc::tmem_ld32(pvrow + c * 32, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[c * 32 + i] = o[c * 32 + i] * corr + v[i];
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&pv_empty[gr]));
      };
      for (int j = gr; j < w.n; j += 2) {
        const uint32_t i0 = it + j, st = i0 % C::kStages, ph = (i0 / C::kStages) & 1;
        const int p0 = (w.t0 + j) * kTile;
        const bool tail = p0 + kTile > base;
        if constexpr (kFp8) {
          // the tile's scales as floats, a token a thread
          ok = ok && mbar_wait(smem_u32(&kfull[st]), ph, &g_err_tree);
          const uint32_t kc = scales[st][0][r], vc = scales[st][1][r];
          float inv = __uint_as_float((254u - vc) << 23);
          if (tail && !(inv >= 0.f && inv < INFINITY)) inv = 0.f;  // stale scale bytes
          named_bar_sync(bar, 128);                                 // the tile before is done with them
          tok_k[gr][r] = __uint_as_float(kc << 23);
          tok_b[gr][r] = (float)((int)vc - 127);
          tok_i[gr][r] = inv;
          named_bar_sync(bar, 128);
        }
        ok = ok && mbar_wait(smem_u32(&s_full[gr]), use & 1, &g_err_tree);
        tc::fence_after();
        // four scores of a row, from token t on, as powers of two
        const auto scores4 = [&](float* s, int t) {
          if constexpr (kFp8) {
            const float4 k = *reinterpret_cast<const float4*>(&tok_k[gr][t]), b = *reinterpret_cast<const float4*>(&tok_b[gr][t]);
            s[0] = fmaf(s[0] * rscale, k.x, b.x);
            s[1] = fmaf(s[1] * rscale, k.y, b.y);
            s[2] = fmaf(s[2] * rscale, k.z, b.z);
            s[3] = fmaf(s[3] * rscale, k.w, b.w);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] *= rscale;
          }
        };
        float mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tc::tmem_ld32(srow + c * 32, v);
#pragma unroll
          for (int i = 0; i < 32; i += 4) scores4(v + i, c * 32 + i);
          if (tail) {
            const uint32_t seen = in ? seen32(a, qrow, node, base, w.s.len, p0 + c * 32) : 0u;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = (seen >> i) & 1u ? v[i] : -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, v[i]);
        }
        const float m_new = fmaxf(m_run, mx);
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float corr = ex2(m_run - ref);
        float psum = 0.f;
        // this group's P was last read by P V of its tile before, folded below
        if (pending) fold(corr_prev);
        corr_prev = corr;
        const float shift = kFp8 ? ref - 8.f : ref;  // e4m3 weights are scaled by 2^8
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tc::tmem_ld32(srow + c * 32, v);
#pragma unroll
          for (int i = 0; i < 32; i += 4) scores4(v + i, c * 32 + i);
          if (tail) {
            const uint32_t seen = in ? seen32(a, qrow, node, base, w.s.len, p0 + c * 32) : 0u;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = (seen >> i) & 1u ? v[i] : -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
#pragma unroll
            for (int y = 0; y < 4; ++y) v[i + y] = ex2(v[i + y] - shift);
            if constexpr (kFp8) {
              const float4 n = *reinterpret_cast<const float4*>(&tok_i[gr][c * 32 + i]);
              psum = fmaf(v[i], n.x, psum);
              psum = fmaf(v[i + 1], n.y, psum);
              psum = fmaf(v[i + 2], n.z, psum);
              psum = fmaf(v[i + 3], n.w, psum);
            } else {
              psum += (v[i] + v[i + 1]) + (v[i + 2] + v[i + 3]);
            }
          }
          if constexpr (kFp8) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) split4(v + 4 * i, hi[i], lo[i]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t at = pbase + r * 128 + (((c * 2 + k) ^ (r & 7)) << 4);
              sts128(at, hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]);
              sts128(at + kPart, lo[4 * k], lo[4 * k + 1], lo[4 * k + 2], lo[4 * k + 3]);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              sts128(pbase + (c >> 1) * kPart + r * 128 + ((((c & 1) * 4 + k) ^ (r & 7)) << 4),
                     pack_bf16(v[8 * k], v[8 * k + 1]), pack_bf16(v[8 * k + 2], v[8 * k + 3]),
                     pack_bf16(v[8 * k + 4], v[8 * k + 5]), pack_bf16(v[8 * k + 6], v[8 * k + 7]));
          }
        }
        if (tail) {
          // Rows of V past the context hold stale bytes (possibly NaN), and drafted
          // rows may be hidden from some query rows: a zero weight does not cancel
          // NaN or infinities. Zero the former; take drafted rows that are not
          // finite out of the tile and add them here, row by row.
          ok = ok && mbar_wait(smem_u32(&vfull[st]), ph, &g_err_tree);
          const uint32_t vr = sbase + C::kRing + st * C::kStage + C::kKV + r * 128;
          bool odd = false;
          if (p0 + r >= base && p0 + r < w.s.len) {
#pragma unroll 1
            for (int c = 0; c < (kFp8 ? 8 : 16); ++c) {
              const uint4 x = lds128(vr + (c >> 3) * kPart + ((c & 7) << 4));  // any order: the whole row is looked at
              const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                odd |= kFp8 ? __vcmpeq4(wd[i] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0
                            : __vcmpeq2(wd[i] & 0x7f807f80u, 0x7f807f80u) != 0;
            }
          }
          if (any_of_barrier(bar, 128, odd)) {
            const uint32_t bits = __ballot_sync(0xffffffffu, odd);
            if (lane == 0) odd_bits[gr][qd] = bits;
            named_bar_sync(bar, 128);
#pragma unroll
            for (int i = 0; i < kHD; ++i) o[i] *= corr;
            corr_prev = 1.f;
#pragma unroll 1
            for (int t = 0; t < kTile; ++t) {
              if (!((odd_bits[gr][t >> 5] >> (t & 31)) & 1u)) continue;  // the same for the whole group
              const uint32_t seen = in ? seen32(a, qrow, node, base, w.s.len, p0 + (t & ~31)) : 0u;
              float x = tmem_ld1(srow + t) * rscale;
              if (kFp8) x = fmaf(x, tok_k[gr][t], tok_b[gr][t]);
              if ((seen >> (t & 31)) & 1u) {
                const float p = ex2(x - shift);
                const uint32_t row = sbase + C::kRing + st * C::kStage + C::kKV + t * 128;
#pragma unroll
                for (int c = 0; c < (kFp8 ? 8 : 16); ++c) {
                  const uint4 y = lds128(row + (c >> 3) * kPart + (((c & 7) ^ (t & 7)) << 4));
                  const uint32_t wd[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    if constexpr (kFp8) {
                      uint32_t h0, h1;
                      e4m3x4_to_half(wd[i], h0, h1);
                      const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                      const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                      float* at = o + c * 16 + i * 4;
                      at[0] += p * f0.x, at[1] += p * f0.y, at[2] += p * f1.x, at[3] += p * f1.y;
                    } else {
                      float* at = o + c * 8 + i * 2;
                      at[0] += p * __uint_as_float(wd[i] << 16);
                      at[1] += p * __uint_as_float(wd[i] & 0xffff0000u);
                    }
                  }
                }
              }
              __syncwarp();
            }
            named_bar_sync(bar, 128);
          }
          if (odd || p0 + r >= w.s.len) {
#pragma unroll
            for (int c = 0; c < (kFp8 ? 8 : 16); ++c) sts128(vr + (c >> 3) * kPart + ((c & 7) << 4), 0u, 0u, 0u, 0u);
          }
        }
        tc::fence_before();
        fence_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&s_empty[gr]));
          mbar_arrive(smem_u32(&p_full[gr]));
        }
        l_run = fmaf(l_run, corr, psum);
        m_run = m_new;
        pending = true;
        ++use;
      }
      if (pending) fold(corr_prev);
      it += w.n;

      // ---------------------------------------------- join the two groups' tiles
      if (!ok) m_run = -INFINITY, l_run = 0.f;
      const uint32_t scratch = sbase + C::kP + r * 512;  // both P buffers: no MMA reads them any more
      named_bar_sync(3, kGroups * 128);                  // both groups' MMAs are over (Q is free as well)
      if (w.n > 1) {
        if (gr == 1) {
          m_other[r] = m_run;
          l_other[r] = l_run;
#pragma unroll
          for (int c = 0; c < 32; ++c)
            sts128(scratch + ((c ^ lane) << 4), __float_as_uint(o[4 * c]), __float_as_uint(o[4 * c + 1]),
                   __float_as_uint(o[4 * c + 2]), __float_as_uint(o[4 * c + 3]));
        }
        named_bar_sync(3, kGroups * 128);
      }
      if (gr == 0) {
        float f0 = 1.f;
        if (w.n > 1) {
          const float m1 = m_other[r], M = fmaxf(m_run, m1);
          f0 = m_run == -INFINITY ? 0.f : ex2(m_run - M);
          const float f1 = m1 == -INFINITY ? 0.f : ex2(m1 - M);
          l_run = l_run * f0 + l_other[r] * f1;
          m_run = M;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const uint4 x = lds128(scratch + ((c ^ lane) << 4));
            o[4 * c] = o[4 * c] * f0 + __uint_as_float(x.x) * f1;
            o[4 * c + 1] = o[4 * c + 1] * f0 + __uint_as_float(x.y) * f1;
            o[4 * c + 2] = o[4 * c + 2] * f0 + __uint_as_float(x.z) * f1;
            o[4 * c + 3] = o[4 * c + 3] * f0 + __uint_as_float(x.w) * f1;
          }
        }
        if (in && w.whole()) {
          const float inv = l_run == 0.f ? 0.f : 1.f / l_run;  // nothing seen: 0
          uint4* op = reinterpret_cast<uint4*>(a.out + (int64_t)qrow * a.o_st + (int64_t)head * a.o_sh);
#pragma unroll
          for (int c = 0; c < 16; ++c)
            op[c] = make_uint4(pack_bf16(o[8 * c] * inv, o[8 * c + 1] * inv), pack_bf16(o[8 * c + 2] * inv, o[8 * c + 3] * inv),
                               pack_bf16(o[8 * c + 4] * inv, o[8 * c + 5] * inv), pack_bf16(o[8 * c + 6] * inv, o[8 * c + 7] * inv));
        } else if (in) {
          const int64_t pr = ((int64_t)blockIdx.x * 2 + w.slot()) * kRows + r;
          float4* dst = reinterpret_cast<float4*>(a.part_o + pr * kHD);
#pragma unroll
          for (int c = 0; c < 32; ++c) dst[c] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          a.part_m[pr] = m_run;
          a.part_l[pr] = l_run;
        }
      }
      named_bar_sync(3, kGroups * 128);  // the P buffers are free again
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

}  // namespace tcore
}  // namespace
}  // namespace kvb
