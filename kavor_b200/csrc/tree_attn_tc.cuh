// The tcgen05 form of the tree attention, for units of many query rows: included
// by tree_attn.cu.
//
// A CTA owns 128 query rows (nodes x query heads of one kv head) and walks the
// context in 128-token tiles: S = Q K^T is a tcgen05.mma chain into TMEM, two
// softmax warpgroups take the tiles in turn (one thread per query row, so no
// reduction crosses threads), walk S twice in loops of 64 columns (straight-line
// code for a row missed the instruction cache) and put the weights P in TMEM, from
// where a second chain adds P V to the output rows, also in TMEM. One group's
// exponentials overlap the other group's and the MMAs. Both groups weigh a row
// against the same reference, settled tile by tile (a barrier hands it from group to
// group); it moves only when a tile's maximum passes it by 2^15: weights of up to
// 2^15 cost nothing in bf16, and the output rows are rescaled once or twice
// in a context instead of at every tile (a rescale waits for the P V before it: with
// 2^8, 16 x 64 nodes over e4m3 took 564 us instead of 465). Loads, MMAs and the
// conversion of V have warps of their own, each waiting for nothing it does not need.
//
// Over an e4m3 cache K stays e4m3: Q is split in two e4m3 parts, x = hi + lo, hi =
// e4m3(x), lo = e4m3(x - hi), which hold a bf16 value (8 bits, two signed 4-bit
// significands) exactly down to 2^-10 of its row's maximum, scaled to [128, 256),
// and to 2^-18 of that maximum below it. Two e4m3 chains take as long as one
// 16-bit chain and K is never converted. V becomes bf16, times its row's scale: four
// warps do that, exactly (four significant bits, every scale that is written), so V's
// scale is in no score and no reference, whatever the rows' sizes are (a zero row is
// held with the scale 2^0: in the scores it raised the reference by up to 2^14). The
// weights are bf16 (2^-8 of each), as over the bf16 cache.
//
// Measured, 64 query heads over 8 kv heads, 16 trees of 64 nodes, 3900 to 8100
// tokens: 278 us over bf16 (724 TFLOP/s; K and V come 3.9 times from HBM, once for each
// of a sequence's row blocks: 5.4 TB/s), 390 over e4m3 (516). A tile takes 2400 clocks
// over bf16, of which the two MMA chains issue for 1170 and the exponentials (16 a
// clock) take 1024. Over e4m3 each score takes K's scale and is stored between the
// walks, V's scaling takes 27 us (363 without), and with these inputs' wide scores a
// tile in five rescales some of its rows.
// 64 trees of 9 to 32 nodes, 32 heads over 8, 200 to 2300 tokens of bf16: 89 us, the
// fixed 10,000 clocks of each of the 512 units beside their 18 tiles at most.
#pragma once

namespace kvb {
namespace {
namespace tcore {

constexpr int kRows = 128;
constexpr int kTile = 128;
constexpr int kGroups = 2;                                // softmax warpgroups
constexpr uint32_t kCols = 512;                           // S0, S1, O: 128 columns each; P0, P1: 64
constexpr uint32_t kColO = 256, kColP = 384;
constexpr float kSlack = 15.f;                            // log2 of the largest weight
constexpr int kHalf = kTile * 128;                        // 128 rows of 128 bytes
constexpr int kOperand = 2 * kHalf;                       // 16-bit Q or V (two halves of 64 dims), or two e4m3 parts of Q
// Warps 0 and 2 load K and V, 1 issues Q K^T, 3 issues P V, 4 to 7 load Q and
// convert V of an e4m3 cache; then the softmax groups.
constexpr int kFirst = 8, kThreads = kFirst * 32 + kGroups * 128;
// Registers: 128 a thread at launch; the other warps give theirs up for the
// softmax threads: 128 (2 * 64 + 2 * 192) = 512 * 128.
constexpr int kOtherRegs = 64, kSoftmaxRegs = 192;
template <bool kFp8>
struct Cfg {
  static constexpr int kKV = kTile * kHD * (kFp8 ? 1 : 2);
  static constexpr int kStages = 3;
  static constexpr int kQ = 0, kV16 = kOperand, kRing = kOperand + (kFp8 ? 2 * kOperand : 0);
  static constexpr int kSmem = kRing + kStages * 2 * kKV + 1024;
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
// The MMAs and commits are written for a whole warp: the instruction itself elects
// its one thread. A warp without a branch keeps the descriptors in uniform
// registers; from one thread's branch each MMA waited 93 cycles for its descriptors'
// way there (an MMA itself takes 64).
template <bool kFp8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (kFp8)
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
  else
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// D (+)= P V with the 16-bit P in TMEM (two values a column, a row a lane).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
// The same value in every lane, known as such to the compiler.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
// The arriving half of a named barrier whose other half waits.
__device__ __forceinline__ void named_bar_arrive(int id, int nthreads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
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
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  return r;
}
// 32 columns of this thread's lane into r[kAt..], without waiting; ready after landed().
template <int kAt, int kN>
__device__ __forceinline__ void tmem_get(uint32_t taddr, float (&v)[kN]) {
  float* r = v + kAt;
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
template <int kAt, int kN>
__device__ __forceinline__ void pin(float (&v)[kN]) {  // no use of the registers moves before this
  float* r = v + kAt;
  asm volatile(""
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                 "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]),
                 "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]),
                 "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31]));
}
// 64 columns of a row.
__device__ __forceinline__ void tmem_row64(uint32_t taddr, float (&v)[64]) {
  tmem_get<0>(taddr, v);
  tmem_get<32>(taddr + 32, v);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  pin<0>(v);
  pin<32>(v);
}
// 16 columns of this thread's lane.
__device__ __forceinline__ void tmem_put16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
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
  __shared__ __align__(8) uint64_t q_full, q_empty, kfull[C::kStages], vfull[C::kStages], k_empty[C::kStages], v_empty[C::kStages],
      v16_full[2], v16_empty[2], s_full[2], s_empty[2], p_full[2], pv_full[2], o_empty;
  __shared__ __align__(16) uint8_t scales[kFp8 ? C::kStages : 1][2][kTile];
  __shared__ __align__(16) float tok_k[kFp8 ? 4 : 1][kTile];  // scales of a tile's K rows; two tiles of each group
  __shared__ float ref_s[kRows], l_s[2][kRows];
  __shared__ float qs_s[kFp8 ? 4 : 1][kRows];  // scale of a query row's e4m3 parts, of four segments
  __shared__ uint32_t o_started;  // the output rows hold something before a segment's first P V
  __shared__ uint32_t odd_bits[2][4];
  __shared__ uint32_t tmem_s;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&q_full), 4);
    mbar_init(smem_u32(&q_empty), 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(smem_u32(&kfull[i]), 1);
      mbar_init(smem_u32(&vfull[i]), 1);
      mbar_init(smem_u32(&k_empty[i]), kFp8 ? 5 : 1);  // the MMAs; the four warps that read K's scales
      mbar_init(smem_u32(&v_empty[i]), kFp8 ? 4 : 1);  // the converting warps, or the MMAs
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&v16_full[i]), 4);
      mbar_init(smem_u32(&v16_empty[i]), 1);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&s_empty[i]), 4);
      mbar_init(smem_u32(&p_full[i]), 4);
      mbar_init(smem_u32(&pv_full[i]), 1);
    }
    mbar_init(smem_u32(&o_empty), kGroups * 4);
    o_started = 0;
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
  // Tile i of the CTA: stage i % kStages of the rings (use i / kStages of it),
  // V buffer i & 1 (use i / 2); tile j of a segment belongs to group j & 1.
  const auto stage_of = [](uint32_t i) { return i % C::kStages; };
  const auto phase_of = [](uint32_t i) { return (i / C::kStages) & 1; };

  if (warp < kFirst) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 0 || warp == 2) {
      // ------------------------------------------------- TMA producers, K and V
      // (in one thread, K waited behind V's buffers, which are held until P V has
      // ended: 16 x 64 nodes over bf16 took 367 us, apart 337)
      const bool do_k = warp == 0, do_v = warp == 2;
      if (lane == 0) {
        prefetch_tensormap(do_k ? &kmap : &vmap);
        const uint64_t pol = l2_evict_first_policy();
        const int boxes = kTile / a.box;
        uint32_t it = 0;
        bool ok = true;
        while (ok && w.next(a)) {
          const bool once = w.s.blocks == 1;  // else several row blocks read the same rows: keep those in L2
          const auto load = [&](const CUtensorMap* map, uint32_t dst, int off, int blk, uint32_t bar) {
#pragma unroll
            for (int hf = 0; hf < (kFp8 ? 1 : 2); ++hf) {
              if (once)
                tma_load_4d(dst + hf * kHalf, map, hf * 64, w.h, off, blk, bar, pol);
              else
                tma_load_4d_keep(dst + hf * kHalf, map, hf * 64, w.h, off, blk, bar);
            }
          };
          tree::Pages pg;
          pg.start(a, w, w.t0 * kTile);
          for (int j = 0; j < w.n && ok; ++j, ++it) {
            const uint32_t st = stage_of(it), kd = sbase + C::kRing + st * 2 * C::kKV, vd = kd + C::kKV;
            const uint32_t kb = smem_u32(&kfull[st]), vb = smem_u32(&vfull[st]);
            if (it >= C::kStages) {
              if (do_k) ok = mbar_wait(smem_u32(&k_empty[st]), phase_of(it - C::kStages), &g_err_tree);
              if (do_v) ok = ok && mbar_wait(smem_u32(&v_empty[st]), phase_of(it - C::kStages), &g_err_tree);
              if (!ok) break;
            }
            for (int x = 0; x < boxes; ++x) {
              const bool none = pg.absent(a, w);
              const int blk = none ? a.num_blocks : pg.blk;  // out of the tensor map: TMA fills zeros
              const uint32_t bar = do_k ? kb : vb;
              uint8_t* sc = &scales[kFp8 ? st : 0][do_k ? 0 : 1][kFp8 ? x * a.box : 0];
              const uint32_t bytes = C::kKV / boxes + (kFp8 && !none ? a.box : 0);  // rows and their scales
              if (kFp8 && none) {  // zeros, of scale 1
                for (int k = 0; k < a.box / 4; ++k) reinterpret_cast<uint32_t*>(sc)[k] = 0x7f7f7f7fu;
                fence_async();  // before a later copy into the same bytes
              }
              if (x + 1 < boxes)
                mbar_expect_tx(bar, bytes);
              else
                mbar_arrive_expect_tx(bar, bytes);
              if (kFp8 && !none) {
                const int64_t so = blk * a.scale_stride + (int64_t)w.h * a.block_size + pg.off;
                bulk_load(smem_u32(sc), (do_k ? a.ks : a.vs) + so, a.box, bar);
              }
              load(do_k ? &kmap : &vmap, (do_k ? kd : vd) + x * a.box * 128, pg.off, blk, bar);
              pg.advance(a, w, a.box);
            }
          }
        }
        if (do_k) w.leave(a);
        // no copy may outlive the CTA: wait (bounded) for the last phase of every stage
        for (uint32_t i = it < C::kStages ? 0 : it - C::kStages; i < it; ++i) {
          if (do_k) mbar_wait(smem_u32(&kfull[stage_of(i)]), phase_of(i), &g_err_tree);
          if (do_v) mbar_wait(smem_u32(&vfull[stage_of(i)]), phase_of(i), &g_err_tree);
        }
      }
    } else if (warp == 1 || warp == 3) {
      // ----------------------------------------------------------- MMA issuers
      // fp32 accumulation, M = N = 128. Q K^T: bf16, or e4m3 parts of Q; P V: bf16,
      // V read head-dim-major (bit 16). A warp for each, so that neither waits behind
      // what the other waits for.
      constexpr uint32_t kShape = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
      constexpr uint32_t kBf16 = (1u << 7) | (1u << 10);
      constexpr int kParts = kFp8 ? 2 : 1, kSteps = kFp8 ? 4 : 8;  // Q K^T: MMAs of 32 or 16 dims
      uint32_t it = 0, seg = 0, done[2] = {0, 0};                  // tiles, segments, tiles of each group so far
      bool ok = true;
      while (ok && w.next(a)) {
        if (warp == 1 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&q_full), seg & 1, &g_err_tree))) break;
        for (int j = 0; j < w.n; ++j) {
          const uint32_t i = it + j, st = stage_of(i), gr = j & 1, use = done[gr] + (j >> 1);
          if (warp == 1) {  // S, once the tile before in its buffer has been weighed
            ok = (use == 0 || mbar_wait(smem_u32(&s_empty[gr]), (use - 1) & 1, &g_err_tree)) &&
                 mbar_wait(smem_u32(&kfull[st]), phase_of(i), &g_err_tree);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc::fence_after();
            const uint64_t q = desc_k(sbase + C::kQ), k = desc_k(uniform(sbase + C::kRing + st * 2 * C::kKV));
            const uint32_t d = uniform(tmem + gr * 128);
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
              for (int ks = 0; ks < kSteps; ++ks) {
                // descriptors count 16 bytes
                const uint32_t off = ((kFp8 ? 0 : (ks >> 2) * kHalf) + (ks & 3) * 32) >> 4;
                mma<kFp8>(d, q + (part * kHalf >> 4) + off, k + off, kShape | (kFp8 ? 0u : kBf16), part > 0 || ks > 0);
              }
            commit(smem_u32(&k_empty[st]));
            if (j == w.n - 1) commit(smem_u32(&q_empty));
            commit(smem_u32(&s_full[gr]));
          } else {
            ok = mbar_wait(smem_u32(kFp8 ? &v16_full[i & 1] : &vfull[st]), kFp8 ? (i >> 1) & 1 : phase_of(i), &g_err_tree) &&
                 // a segment's first P V overwrites the output rows of the segment before
                 (j > 0 || seg == 0 || mbar_wait(smem_u32(&o_empty), (seg - 1) & 1, &g_err_tree)) &&
                 mbar_wait(smem_u32(&p_full[gr]), use & 1, &g_err_tree);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc::fence_after();
            const uint64_t v =
                desc_mn(uniform(sbase + (kFp8 ? C::kV16 + (i & 1) * kOperand : C::kRing + st * 2 * C::kKV + C::kKV)), kHalf);
            const uint32_t more = uniform(j > 0 || *reinterpret_cast<volatile uint32_t*>(&o_started));
            const uint32_t d = uniform(tmem + kColO), p = uniform(tmem + kColP + gr * 64);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              mma_ts(d, p + ks * 8, v + ks * (2048 >> 4), kShape | kBf16 | (1u << 16), ks > 0 ? 1u : more);
            commit(smem_u32(kFp8 ? &v16_empty[i & 1] : &v_empty[st]));
            commit(smem_u32(&pv_full[gr]));
          }
        }
        it += w.n;
        ++seg;
        done[0] += (w.n + 1) >> 1;
        done[1] += w.n >> 1;
      }
    } else {
      // --------------------------- query rows; V's e4m3 bytes and scales to bf16
      uint32_t it = 0;
      bool ok = true;
      const int t2 = threadIdx.x - 128;
      for (uint32_t seg = 0; w.next(a); ++seg) {
        // half a warp a row, rows 8 apart, once the last segment's Q K^T has read
        // the rows before. (Read by the softmax threads, each its row, a segment
        // began 20,000 to 27,000 cycles after the last tile of the one before.)
        ok = ok && (seg == 0 || mbar_wait(smem_u32(&q_empty), (seg - 1) & 1, &g_err_tree));
        const int c = t2 & 15;
#pragma unroll 1
        for (int r0 = t2 >> 4; r0 < kRows; r0 += 32) {
          uint4 x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t R = w.rb * kRows + r0 + i * 8, node = R / (uint32_t)a.group;
            const int head = w.h * a.group + (int)(R - node * a.group);
            const bool in = node < (uint32_t)w.s.nodes;
            const bf16* src = a.q + (int64_t)(w.s.q0 + (in ? node : 0)) * a.q_st + (int64_t)head * a.q_sh + c * 8;
            if constexpr (kFp8) {
              x[i] = make_uint4(0u, 0u, 0u, 0u);
              if (in) x[i] = *reinterpret_cast<const uint4*>(src);
            } else {
              const int row = r0 + i * 8;
              copy16(sbase + C::kQ + (c >> 3) * kHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4), src, in);
            }
          }
          if constexpr (kFp8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = r0 + i * 8;
              const uint32_t wd[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
              uint32_t mx = 0, inf = 0;
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint32_t z = wd[y] & 0x7fff7fffu, big = __vcmpgtu2(z, 0x7f7f7f7fu);
                inf |= big;
                mx = __vmaxu2(mx, z & ~big);
              }
              mx = max(mx & 0xffffu, mx >> 16);
#pragma unroll
              for (int o = 1; o < 16; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
              const bool odd = (__ballot_sync(0xffffffffu, inf != 0) >> (lane & 16) & 0xffffu) != 0;
              const int e = max((int)(mx >> 7) - 127 - 7, -126);  // the largest to [128, 256), to 1 at least
              const float inv = pow2(-e);
              float f[8];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&wd[y]));
                f[2 * y] = v.x * inv;
                f[2 * y + 1] = v.y * inv;
              }
              uint2 hi, lo;
              split4(f, hi.x, lo.x);
              split4(f + 4, hi.y, lo.y);
              uint8_t* at = smem + C::kQ + row * 128 + (((c >> 1) ^ (row & 7)) << 4) + (c & 1) * 8;
              *reinterpret_cast<uint2*>(at) = hi;
              *reinterpret_cast<uint2*>(at + kHalf) = lo;
              // A row with NaN or an infinity gives NaN. The softmax threads have this by S,
              // those of segment seg - 4 are done: the Q K^T of seg - 1 that ended waited for
              // a tile of seg - 2, weighed after the barrier at the end of seg - 3
              if (c == 0) qs_s[seg & 3][row] = odd ? NAN : a.scale_log2 * pow2(e);
            }
          }
        }
        if constexpr (!kFp8) copies_done();
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&q_full));
        for (int j = 0; kFp8 && j < w.n; ++j, ++it) {
          const uint32_t st = stage_of(it), buf = it & 1;
          ok = ok && mbar_wait(smem_u32(&vfull[st]), phase_of(it), &g_err_tree) &&
               (it < 2 || mbar_wait(smem_u32(&v16_empty[buf]), ((it >> 1) - 1) & 1, &g_err_tree));
          if (!ok) continue;
          const uint32_t src = sbase + C::kRing + st * 2 * C::kKV + C::kKV, dst = sbase + C::kV16 + buf * kOperand;
#pragma unroll 4
          for (int i = 0; i < 8; ++i) {
            // 16 dims (chunk c) of token t: two 8-dim chunks of its row's half c / 4
            const int idx = i * 128 + t2, t = idx >> 3, c = idx & 7;
            const uint4 x = lds128(src + t * 128 + ((c ^ (t & 7)) << 4));
            const float vsc = __uint_as_float((uint32_t)scales[st][1][t] << 23);
            const uint64_t v2 = pk2(vsc, vsc);
            uint32_t y[8];
            e4m3x4_to_half(x.x, y[0], y[1]);
            e4m3x4_to_half(x.y, y[2], y[3]);
            e4m3x4_to_half(x.z, y[4], y[5]);
            e4m3x4_to_half(x.w, y[6], y[7]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y[k]));
              float f0, f1;
              un2(mul2(pk2(f.x, f.y), v2), f0, f1);
              y[k] = pack_bf16(f0, f1);
            }
            const uint32_t row = dst + (c >> 2) * kHalf + t * 128;
            const int first = (c & 3) * 2, odd = c >> 2;  // the halves' lanes start on different banks
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const bool up = (k ^ odd) != 0;
              sts128(row + (((first + up) ^ (t & 7)) << 4), up ? y[4] : y[0], up ? y[5] : y[1], up ? y[6] : y[2],
                     up ? y[7] : y[3]);
            }
          }
          fence_async();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(&v16_full[buf]));
            mbar_arrive(smem_u32(&v_empty[st]));
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------ softmax groups
    // A wait that gave up (its error bit is set) is not followed by others, and the
    // group goes on with what is there: its barriers stay matched, its rows are dropped.
    const int gr = (warp - kFirst) >> 2;                  // group: tiles of its parity
    const int qd = warp & 3;                         // TMEM lane quarter of this warp
    const int r = qd * 32 + lane;                    // query row of the unit = TMEM lane; token of a tile
    const int bar = 1 + gr;                          // the group's named barrier
    const uint32_t lane_base = tmem + ((uint32_t)(qd * 32) << 16);
    const uint32_t srow = lane_base + gr * 128, orow = lane_base + kColO, prow = lane_base + kColP + gr * 64;
    uint32_t it = 0, use = 0, other = 0;  // tiles of the CTA, of this group, of the other group in the segments before
    bool ok = true;
    uint32_t seg = 0;
    for (; w.next(a); ++seg) {
      const int base = w.s.len - w.s.nodes;
      const int R = w.rb * kRows + r, node = R / a.group;
      const bool in = node < w.s.nodes;
      const int qrow = w.s.q0 + (in ? node : 0);
      const int head = w.h * a.group + (in ? R - node * a.group : 0);
      float rscale = a.scale_log2;

      float m_ref = -INFINITY, l_run = 0.f;
      // until P V of this group's tile k, or the other group's, has ended
      const auto wait_pv = [&](uint32_t k) {
        ok = ok && mbar_wait(smem_u32(&pv_full[gr]), k & 1, &g_err_tree);
        tc::fence_after();
      };
      const auto wait_pv_other = [&](uint32_t k) {
        ok = ok && mbar_wait(smem_u32(&pv_full[gr ^ 1]), k & 1, &g_err_tree);
        tc::fence_after();
      };
      const uint32_t use0 = use;
      for (int j = gr; j < w.n; j += 2) {
        const uint32_t i0 = it + j, st = stage_of(i0), tb = gr * 2 + (use & 1);
        const int p0 = (w.t0 + j) * kTile;
        const bool tail = p0 + kTile > base;
        if constexpr (kFp8) {
          // K's scales of the tile as floats, a token a thread (the buffer's last
          // readers have passed the barrier of the tile between)
          ok = ok && mbar_wait(smem_u32(&kfull[st]), phase_of(i0), &g_err_tree);
          tok_k[tb][r] = __uint_as_float((uint32_t)scales[st][0][r] << 23);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&k_empty[st]));
          named_bar_sync(bar, 128);
        }
        uint32_t seen[4];
        if (tail)
#pragma unroll
          for (int i = 0; i < 4; ++i) seen[i] = in ? seen32(a, qrow, node, base, w.s.len, p0 + i * 32) : 0u;
        ok = ok && mbar_wait(smem_u32(&s_full[gr]), use & 1, &g_err_tree);
        tc::fence_after();
        if constexpr (kFp8) rscale = qs_s[seg & 3][r];
        // first walk: the tile's scores, as powers of two (bf16: times the row's
        // scale in the second walk), back to S where that saves the second walk
        // something, and their maximum
        const uint64_t rs2 = pk2(rscale, rscale);
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          float v[64];
          tmem_row64(srow + c, v);
          if constexpr (kFp8) {
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
              const float4 k = *reinterpret_cast<const float4*>(&tok_k[tb][c + i]);
              un2(mul2(pk2(v[i], v[i + 1]), mul2(rs2, pk2(k.x, k.y))), v[i], v[i + 1]);
              un2(mul2(pk2(v[i + 2], v[i + 3]), mul2(rs2, pk2(k.z, k.w))), v[i + 2], v[i + 3]);
            }
          }
          if (tail) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t bits = c == 0 ? seen[h] : seen[2 + h];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[h * 32 + i] = (bits >> i) & 1u ? v[h * 32 + i] : -INFINITY;
            }
          }
#pragma unroll
          for (int i = 0; i < 64; i += 8)
#pragma unroll
            for (int y = 0; y < 4; ++y) mx[y] = fmaxf(mx[y], fmaxf(v[i + 2 * y], v[i + 2 * y + 1]));
          if (kFp8 || tail) {
            tc::tmem_st32(srow + c, v);
            tc::tmem_st32(srow + c + 32, v + 32);
          }
        }
        float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (!kFp8) m_tile *= rscale;
        // the row's reference, as the tile before left it
        if (j > 0) {
          named_bar_sync(4 + (gr ^ 1), kGroups * 128);
          const float left = ref_s[r];
          if (left != m_ref) {
            l_run *= m_ref == -INFINITY ? 0.f : ex2(m_ref - left);  // keeps NaN
            m_ref = left;
          }
        }
        const bool move = j == 0 || m_tile > m_ref + kSlack;
        if (__any_sync(0xffffffffu, move)) {
          const float m_new = move ? fmaxf(m_ref, m_tile) : m_ref;
          if (j > 0) {
            const float corr = m_new == m_ref ? 1.f : ex2(m_ref - m_new);
            wait_pv_other(other + ((j + 1) >> 1) - 1);  // the tile before: P V run in order
#pragma unroll 1
            for (int c = 0; c < 128; c += 64) {
              float y[64];
              tmem_row64(orow + c, y);
#pragma unroll
              for (int i = 0; i < 64; ++i) y[i] *= corr;
              tc::tmem_st32(orow + c, y);
              tc::tmem_st32(orow + c + 32, y + 32);
            }
            l_run *= corr;
          }
          m_ref = m_new;
        }
        if (j + 1 < w.n) {
          ref_s[r] = m_ref;
          named_bar_arrive(4 + gr, kGroups * 128);
        }
        const float ref = m_ref == -INFINITY ? 0.f : m_ref;
        if (use > use0) wait_pv(use - 1);  // this group's P was read by P V of its tile before
        uint64_t sum[4] = {0, 0, 0, 0};
        const uint64_t nref = pk2(-ref, -ref);
        // second walk: the weights
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          float v[64];
          tmem_row64(srow + c, v);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t p[16];
#pragma unroll
            for (int i = h * 32; i < h * 32 + 32; i += 8) {
              uint64_t e[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint64_t s2 = pk2(v[i + 2 * y], v[i + 2 * y + 1]);
                float x0, x1;
                un2(kFp8 ? add2(s2, nref) : fma2(s2, rs2, nref), x0, x1);
                x0 = ex2(x0);
                x1 = ex2(x1);
                p[(i & 31) / 2 + y] = pack_bf16(x0, x1);
                e[y] = pk2(x0, x1);
              }
#pragma unroll
              for (int y = 0; y < 4; ++y) sum[y] = add2(sum[y], e[y]);
            }
            tmem_put16(prow + c / 2 + h * 16, p);
          }
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&s_empty[gr]));
        {
          const uint64_t x = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
          float s0, s1;
          un2(x, s0, s1);
          l_run += s0 + s1;
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        if (tail) {
          // Rows of V past the context hold stale bytes (possibly NaN), and drafted
          // rows may be hidden from some query rows: a zero weight does not cancel
          // NaN or infinities. Zero the former; take drafted rows that are not
          // finite out of the tile and add their share, summed here row by row, to the
          // output rows, before the tile's own P V.
          ok = ok && mbar_wait(smem_u32(kFp8 ? &v16_full[i0 & 1] : &vfull[st]), kFp8 ? (i0 >> 1) & 1 : phase_of(i0),
                               &g_err_tree);
          const uint32_t vt = sbase + (kFp8 ? C::kV16 + (i0 & 1) * kOperand : C::kRing + st * 2 * C::kKV + C::kKV);
          const uint32_t vr = vt + r * 128;
          bool odd = false;
          if (p0 + r >= base && p0 + r < w.s.len) {
#pragma unroll 4
            for (int c = 0; c < 16; ++c) {
              // the whole row is looked at, so any order will do: one that starts each lane on other banks
              const int k = (c + r) & 15;
              const uint4 x = lds128(vr + (k >> 3) * kHalf + ((k & 7) << 4));
              constexpr uint32_t ex = 0x7f807f80u;
              odd |= (__vcmpeq2(x.x & ex, ex) | __vcmpeq2(x.y & ex, ex) | __vcmpeq2(x.z & ex, ex) |
                      __vcmpeq2(x.w & ex, ex)) != 0;
            }
          }
          if (any_of_barrier(bar, 128, odd)) {
            const uint32_t bits = __ballot_sync(0xffffffffu, odd);
            if (lane == 0) odd_bits[gr][qd] = bits;
            named_bar_sync(bar, 128);
            if (j > 0) wait_pv_other(other + ((j + 1) >> 1) - 1);
#pragma unroll 1
            for (int d = 0; d < 4; ++d) {  // 32 dims at a time: few registers beside the main path's
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
#pragma unroll 1
              for (int t = 0; t < kTile; ++t) {
                if (!((odd_bits[gr][t >> 5] >> (t & 31)) & 1u)) continue;  // the same for the whole group
                const uint32_t bits = t < 64 ? t < 32 ? seen[0] : seen[1] : t < 96 ? seen[2] : seen[3];
                const uint32_t two = tmem_ld1(prow + (t >> 1)) >> (t & 1 ? 16 : 0);
                if ((bits >> (t & 31)) & 1u) {
                  const float p = __uint_as_float(two << 16);
#pragma unroll
                  for (int c = 0; c < 4; ++c) {
                    const uint4 y = lds128(vt + t * 128 + (d >> 1) * kHalf + ((((d & 1) * 4 + c) ^ (t & 7)) << 4));
                    const uint32_t wd[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&wd[i]));
                      v[c * 8 + i * 2] += p * f.x;
                      v[c * 8 + i * 2 + 1] += p * f.y;
                    }
                  }
                }
                __syncwarp();
              }
              float y[32];
              if (j > 0) tc::tmem_ld32(orow + d * 32, y);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += j > 0 ? y[i] : 0.f;
              tc::tmem_st32(orow + d * 32, v);
            }
            if (j == 0 && r == 0) o_started = 1;
            named_bar_sync(bar, 128);
          }
          if (odd || p0 + r >= w.s.len) {
#pragma unroll 4
            for (int c = 0; c < 16; ++c) {
              const int k = (c + r) & 15;
              sts128(vr + (k >> 3) * kHalf + ((k & 7) << 4), 0u, 0u, 0u, 0u);
            }
          }
          fence_async();
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[gr]));
        ++use;
      }

      // ------------------------------- the segment's rows: 64 dims for each group
      const bool had_last = ((w.n - 1) & 1) == gr;
      other += gr == 0 ? w.n >> 1 : (w.n + 1) >> 1;
      if (had_last) {
        wait_pv(use - 1);
        ref_s[r] = m_ref;
      } else {
        wait_pv_other(other - 1);
      }
      it += w.n;
      named_bar_sync(3, kGroups * 128);  // every tile of both groups is done
      const float m_end = ref_s[r];
      l_s[gr][r] = l_run * (m_ref == -INFINITY ? 0.f : ex2(m_ref - m_end));  // keeps NaN
      if (threadIdx.x == kFirst * 32) o_started = 0;
      float o[64];
      {
        float y[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tc::tmem_ld32(orow + gr * 64 + c * 32, y);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[c * 32 + i] = y[i];
        }
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&o_empty));
      named_bar_sync(3, kGroups * 128);
      const float l_end = ok ? l_s[0][r] + l_s[1][r] : 0.f;
      if (in) {
        if (w.whole()) {
          const float inv = l_end == 0.f ? 0.f : 1.f / l_end;  // nothing seen: 0
          uint4* op = reinterpret_cast<uint4*>(a.out + (int64_t)qrow * a.o_st + (int64_t)head * a.o_sh + gr * 64);
#pragma unroll
          for (int c = 0; c < 8; ++c)
            op[c] = make_uint4(pack_bf16(o[8 * c] * inv, o[8 * c + 1] * inv), pack_bf16(o[8 * c + 2] * inv, o[8 * c + 3] * inv),
                               pack_bf16(o[8 * c + 4] * inv, o[8 * c + 5] * inv), pack_bf16(o[8 * c + 6] * inv, o[8 * c + 7] * inv));
        } else {
          const int64_t pr = ((int64_t)blockIdx.x * 2 + w.slot()) * kRows + r;
          // four dims of 128 rows together: a warp's stores fill whole lines
          float4* dst = reinterpret_cast<float4*>(a.part_o + (pr - r) * kHD) + gr * 16 * kRows + r;
#pragma unroll
          for (int c = 0; c < 16; ++c)
            dst[c * kRows] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          if (gr == 0) {
            a.part_m[pr] = ok ? m_end : -INFINITY;
            a.part_l[pr] = l_end;
          }
        }
      }
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
