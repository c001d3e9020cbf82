// Work partition shared by the tree-attention kernels and their merge.
//
// A unit is one (sequence, group of kv heads, block of query rows of each): it
// walks the sequence's context in tiles of tokens. The tiles of all units, each unit's
// after kLead more for its fixed cost, in the order sequence > head group > row
// block, form one line that is cut into ranges of equal length, one per CTA (at most
// `parts`): every CTA has about the same work whatever the lengths of the sequences
// are, and the host needs none of the device's lengths. A unit cut between CTAs leaves fp32
// partials (unnormalised rows, running maximum and sum) that the merge joins
// in order, so results do not depend on timing. Included by tree_attn.cu after
// its error word.
#pragma once

#include "common.cuh"

namespace kvb {
namespace tree {

constexpr int kHD = 128;
// What a unit costs besides its tiles (queries, first loads, output), in tiles: it
// lies on the line before its first tile. With 0, 2, 4 and 6, us: 64 trees of 9 to 32
// nodes over 200 to 2300 tokens of bf16 118, 96, 89, 90; decode of 256 over 50 to 2000
// tokens of bf16 227, 188 (3), 176, 177; of e4m3 106, 103 (2), 104, 105; 16 x 64 nodes
// over e4m3 434, 427, 423, 421.
constexpr int kLead = 4;

struct Args {
  const bf16* q;
  int64_t q_st, q_sh;
  int64_t total_q;
  const int32_t* tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* ctx;
  const int32_t* cu_q;
  const uint32_t* mask;  // visibility words of each node, NULL: causal chain
  int64_t mask_stride;
  int mask_words;
  bf16* out;
  int64_t o_st, o_sh;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t scale_stride;  // bytes between blocks of the scale arrays
  int batch, hq, hkv, group;
  int num_blocks, block_size;
  int heads;              // kv heads of a unit
  int head_groups;        // groups of that many
  int row_shift, tile_shift;  // rows and tile are powers of two
  int parts, rows, tile;  // CTAs of the attention grid, query rows of a unit and head, tokens of a tile
  int box;                // tokens of a TMA box: a tile's, or a page's when that is smaller
  int by_dims;            // partials by dims: [parts][2][32][rows][4] (heads = 1)
  float* part_o;          // [parts][2][heads][rows][128]
  float* part_m;          // [parts][2][heads][rows]
  float* part_l;
  struct Cut* cuts;       // [parts]: the unit each part leaves unfinished, written for the merge
  float scale_log2;
};

// A unit that begins in a part and goes on in the next ones.
struct alignas(16) Cut {
  int n;         // parts that hold a piece of it; 0: no such unit
  int rows;      // its query rows for each head
  int q0, row0;  // first query row of the sequence, the unit's first row (nodes x heads of a kv head)
  int h, pad[3];
};

struct Seq {
  int q0, nodes, len;  // first query row, drafted nodes, tokens in the cache (the nodes included)
  int tiles, blocks;   // tiles of the context, row blocks
};

// Sequence b of the batch. Lengths the other arguments cannot serve raise an
// error bit and are cut: a context to its block table, rows outside the query
// tensor to none.
__device__ __forceinline__ Seq seq_of(const Args& a, int b, bool report) {
  Seq s;
  s.q0 = a.cu_q[b];
  const int64_t end = a.cu_q[b + 1];
  s.len = max(a.ctx[b], 0);
  if (s.q0 < 0 || end < s.q0 || end > a.total_q) {
    if (report) atomicOr(&g_err_tree, (unsigned)kErrConfig);
    s.nodes = 0;
  } else {
    s.nodes = (int)(end - s.q0);
  }
  const int64_t room = (int64_t)a.max_blocks * a.block_size;
  if (s.len > room) {
    if (report) atomicOr(&g_err_tree, (unsigned)kErrBlockTable);
    s.len = (int)room;
  }
  s.tiles = (s.len + a.tile - 1) >> a.tile_shift;
  s.blocks = (int)(((int64_t)s.nodes * a.group + a.rows - 1) >> a.row_shift);
  return s;
}
__device__ __forceinline__ int64_t cost_of(const Args& a, const Seq& s) {
  return s.tiles ? (int64_t)(s.tiles + kLead) * s.blocks * a.head_groups : 0;
}

// Exclusive prefix of each thread's sum over the block, and the total.
template <int kThreads>
__device__ __forceinline__ int64_t block_prefix(int64_t mine, int64_t* total) {
  __shared__ int64_t warp_sums[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  *total = all;
  return before + incl - mine;
}

// Length of a range; part p holds [p * range, (p + 1) * range) of the line.
__device__ __forceinline__ int64_t range_of(int64_t total, int parts) {
  // 32 bits are nearly always enough: a 64-bit division takes ten times as long
  return total <= INT32_MAX ? ((uint32_t)total + parts - 1) / (uint32_t)parts : (total + parts - 1) / parts;
}

// Where this CTA's range starts: the sequence, the offset in its tiles, and
// how many tiles the range has. Every thread of the block calls it.
struct Start {
  int b;
  int64_t off, left;
};
template <int kThreads>
__device__ __forceinline__ Start find_start(const Args& a, int part) {
  __shared__ Start s_start;
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(threadIdx.x * per, a.batch), b1 = min(b0 + per, a.batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += cost_of(a, seq_of(a, b, part == 0));
  int64_t total;
  int64_t at = block_prefix<kThreads>(mine, &total);
  const int64_t range = range_of(total, a.parts), lo = range * part, hi = min(lo + range, total);
  if (threadIdx.x == 0) s_start = Start{0, 0, 0};
  __syncthreads();
  if (lo < hi && at <= lo && lo < at + mine) {
    for (int b = b0; b < b1; ++b) {
      const int64_t c = cost_of(a, seq_of(a, b, false));
      if (at <= lo && lo < at + c) s_start = Start{b, lo - at, hi - lo};
      at += c;
    }
  }
  __syncthreads();
  return s_start;
}

// Walks a range segment by segment; a segment is the part of one unit inside it.
struct Walk {
  int b;
  int64_t off, left, range;
  Seq s;
  int h, rb, t0, n;  // first kv head, row block, first tile, tiles
  int rest;          // tiles of the unit after these

  __device__ __forceinline__ Walk(const Args& a, const Start& st) : b(st.b), off(st.off), left(st.left), range(st.left), t0(1) {
    if (left > 0) s = seq_of(a, b, false);
  }
  __device__ __forceinline__ bool next(const Args& a) {
    if (left <= 0) return false;
    for (;;) {
      while (off >= cost_of(a, s)) {
        off = 0;
        if (++b >= a.batch) return false;
        s = seq_of(a, b, false);
      }
      const int len = s.tiles + kLead;
      int64_t u;
      int hg;
      if (off <= UINT32_MAX) {  // nearly always: a 64-bit division takes ten times as long
        u = (uint32_t)off / (uint32_t)len;
        hg = (int)((uint32_t)u / (uint32_t)s.blocks);
      } else {
        u = off / len;
        hg = (int)(u / s.blocks);
      }
      const int pos = (int)(off - u * len), room = len - pos, take = (int)(left < room ? left : room);
      off += take;
      left -= take;
      rest = room - take;
      h = hg * a.heads;
      rb = (int)(u - (int64_t)hg * s.blocks);
      t0 = max(pos - kLead, 0);
      n = max(pos + take - kLead, 0) - t0;
      if (n > 0) return true;
      t0 = 1;  // the range ends before the unit's first tile
      if (left <= 0) return false;
    }
  }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && n == s.tiles; }
  // After the last segment, by one thread of the part.
  __device__ __forceinline__ void leave(const Args& a) const {
    Cut c = {};
    if (t0 == 0 && n < s.tiles) {  // a range that ends inside a unit is a full one
      c.n = 1 + (int)((rest + range - 1) / range);
      c.row0 = rb * a.rows;
      c.rows = min(a.rows, s.nodes * a.group - c.row0);
      c.q0 = s.q0;
      c.h = h;
    }
    a.cuts[blockIdx.x] = c;
  }
  // partial slot of a cut segment: 0 when the unit began in an earlier CTA
  __device__ __forceinline__ int slot() const { return t0 > 0 ? 0 : 1; }
};

// A sequence's pages in order: the page of the current tokens and, loaded ahead,
// the next one (a table entry takes hundreds of cycles to arrive).
struct Pages {
  int col, off;   // page and token in it
  int blk, next;  // block ids; -1 past the context

  __device__ __forceinline__ static int entry(const Args& a, const Walk& w, int col) {
    return (int64_t)col * a.block_size < w.s.len ? a.tables[(int64_t)w.b * a.bt_stride + col] : -1;
  }
  __device__ __forceinline__ void start(const Args& a, const Walk& w, int token) {
    col = token / a.block_size;
    off = token - col * a.block_size;
    blk = entry(a, w, col);
    next = entry(a, w, col + 1);
  }
  __device__ __forceinline__ void advance(const Args& a, const Walk& w, int tokens) {  // tokens divide a page
    off += tokens;
    if (off >= a.block_size) {
      off = 0;
      ++col;
      blk = next;
      next = entry(a, w, col + 1);
    }
  }
  // Nothing to read: past the context, or a block id outside the pool, which raises the error bit.
  __device__ __forceinline__ bool absent(const Args& a, const Walk& w) const {
    if (blk >= 0 && blk < a.num_blocks) return false;
    if ((int64_t)col * a.block_size < w.s.len) atomicOr(&g_err_tree, (unsigned)kErrBlockTable);
    return true;
  }
};

// Does node i of a sequence see node j?
__device__ __forceinline__ bool sees(const Args& a, int row, int i, int j) {
  if (!a.mask) return j <= i;
  const int w = j >> 5;
  return w < a.mask_words && (a.mask[(int64_t)row * a.mask_stride + w] >> (j & 31)) & 1u;
}

}  // namespace tree
}  // namespace kvb
