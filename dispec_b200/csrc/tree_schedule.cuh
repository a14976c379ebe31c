// How the attention of drafted trees is cut among CTAs, shared by its kernels.
//
// Tree s has n_s nodes behind ctx_s stored tokens.  An item is one tile of query rows (rows are (node, head-in-group)
// pairs, G heads a node) of one key/value head of one tree; it walks the key tiles from the first key that any of its
// tree's nodes sees to the tree's last node.  A unit is one key tile of one item.  All units, in the order (tree, head,
// row tile, key tile), are cut into equal runs, one per CTA, wherever that falls: trees of any lengths load every SM
// alike, and nothing about lengths is needed on the host.  Row tiles of one head follow one another, so CTAs that run
// at the same time share its keys through the L2.
//
// An item that ends in the CTA it began in is finished there.  The others leave one partial result (32-bit sums that are
// not divided yet, running maximum, sum of weights) per CTA in scratch: slot 2 c + 1 for the item that begins in CTA c,
// slot 2 c for the one that began before; tree_combine_kernel merges them in the order of the CTAs.
#pragma once
#include "common.cuh"

namespace tree {

struct Shape {
  const int* node_start;  // [S + 1] first row of each tree's nodes
  const int* ctx_len;     // [S] tokens stored in front of the tree
  int S, KVH, G, rows_per_tile, keys_per_tile, window, min_units;
};

// One tree: sizes in units.
struct Tree {
  int first, n, ctx;      // first row, nodes, stored tokens
  int lo_tile, key_tiles; // first key tile any node sees, key tiles from there
  int row_tiles;
};

__device__ __forceinline__ Tree load_tree(const Shape& sh, int s) {
  Tree t;
  t.first = sh.node_start[s];
  t.n = max(0, sh.node_start[s + 1] - t.first);
  t.ctx = max(0, sh.ctx_len[s]);
  // the root sees furthest back: keys from ctx - window + 1
  const int lo = sh.window > 0 ? max(0, t.ctx - sh.window + 1) : 0;
  t.lo_tile = lo / sh.keys_per_tile;
  t.key_tiles = t.n > 0 ? (t.ctx + t.n + sh.keys_per_tile - 1) / sh.keys_per_tile - t.lo_tile : 0;
  t.row_tiles = (int)(((long)t.n * sh.G + sh.rows_per_tile - 1) / sh.rows_per_tile);
  return t;
}
__device__ __forceinline__ long units_of(const Shape& sh, const Tree& t) {
  return (long)t.row_tiles * t.key_tiles * sh.KVH;
}

__device__ __forceinline__ long warp_scan(long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// Units a CTA takes: the same number for all, at least min_units.  Called by whole warps.
__device__ __forceinline__ long units_per_cta(const Shape& sh, int ctas, long* total) {
  const int lane = threadIdx.x & 31;
  long mine = 0;
  for (int s = lane; s < sh.S; s += 32) mine += units_of(sh, load_tree(sh, s));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  *total = mine;
  return max((mine + ctas - 1) / ctas, (long)sh.min_units);
}

// Where unit u lies.
struct Place {
  int seq, item, key_tile;  // item inside the tree: head * row_tiles + row tile; key tile counted from lo_tile
  long item_start;          // first unit of the item
};

// Called by whole warps; u is inside the total.
__device__ __forceinline__ Place find_unit(const Shape& sh, long u) {
  const int lane = threadIdx.x & 31;
  Place p = {0, 0, 0, 0};
  long before = 0;
  for (int s0 = 0; s0 < sh.S; s0 += 32) {
    const int s = s0 + lane;
    Tree t = {};
    long n = 0;
    if (s < sh.S) {
      t = load_tree(sh, s);
      n = units_of(sh, t);
    }
    const long upto = before + warp_scan(n);
    const uint32_t past = __ballot_sync(0xffffffffu, upto > u);
    if (past != 0u) {
      const int who = __ffs(past) - 1;
      const long start = __shfl_sync(0xffffffffu, upto - n, who);
      const int per_item = __shfl_sync(0xffffffffu, t.key_tiles, who);
      p.seq = s0 + who;
      p.item = (int)((u - start) / per_item);
      p.key_tile = (int)((u - start) - (long)p.item * per_item);
      p.item_start = start + (long)p.item * per_item;
      return p;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return p;
}

// A CTA's walk over its run of units, one item's share at a time.
struct Walk {
  long u, end, chunk;
  Place at;
  Tree t;
  // the current share
  int head, row_tile, kt_begin, kt_end;  // key tiles counted from key 0
  int slot;                              // scratch slot of the partial result, -1: the item is finished here

  // false: this CTA has no work
  __device__ __forceinline__ bool begin(const Shape& sh, int cta, int ctas) {
    long total;
    chunk = units_per_cta(sh, ctas, &total);
    u = chunk * cta;
    end = min(total, u + chunk);
    if (u >= end) return false;
    at = find_unit(sh, u);
    t = load_tree(sh, at.seq);
    share(cta);
    return true;
  }
  __device__ __forceinline__ void share(int cta) {
    head = at.item / t.row_tiles;
    row_tile = at.item - head * t.row_tiles;
    const long item_end = at.item_start + t.key_tiles;
    const long stop = min(end, item_end);
    kt_begin = t.lo_tile + at.key_tile;
    kt_end = kt_begin + (int)(stop - u);
    slot = at.key_tile == 0 ? (stop == item_end ? -1 : 2 * cta + 1) : 2 * cta;
  }
  __device__ __forceinline__ bool next(const Shape& sh, int cta) {
    u += kt_end - kt_begin;
    if (u >= end) return false;
    at.key_tile = 0;
    at.item_start = u;
    if (++at.item == t.row_tiles * sh.KVH) {
      at.item = 0;
      do {
        ++at.seq;
        t = load_tree(sh, at.seq);
      } while (t.n == 0);
    }
    share(cta);
    return true;
  }
};

}  // namespace tree

// Merges the partial results of the items that several CTAs share (tree_attn.cu).  part_o: [slot][rows_per_tile][D],
// part_ml: [slot][rows_per_tile] of (maximum in the base-2 domain, sum).
cudaError_t tree_combine(const tree::Shape& sh, const float* part_o, const float* part_ml, void* out, long out_stride,
                         int D, int ctas, int dtype, cudaStream_t stream);
