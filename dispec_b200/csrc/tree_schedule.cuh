// How the attention of drafted trees is cut among CTAs, shared by its kernels.
//
// Tree s has n_s nodes behind ctx_s stored tokens.  An item is one tile of query rows (rows are (node, head-in-group)
// pairs, G heads a node) of one key/value head of one tree; it walks the key tiles from the first key that any of its
// tree's nodes sees to the tree's last node.  A unit is one key tile of one item.  All units, in the order (row tile, tree,
// head, key tile), are cut into equal runs, one per CTA, wherever that falls: trees of any lengths load every SM alike, and
// nothing about lengths is needed on the host.  Where all trees have R row tiles, each row tile's runs are cut alike and
// the CTAs c, c + ctas / R, ... walk the same keys at the same time, which then come from memory once and from the L2
// for the others (64 trees of 320 rows, whose row tiles followed one another in one CTA: 1.28 GB read where
// the keys and values are 0.42).
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
  int S, KVH, G, window, min_units;
  int rows;       // of the queries: a tree that is not inside them is recorded and has no nodes
  int most_ctx;   // tokens that a request's pages hold: more are not stored (their places have no page, which is recorded there)
  int row_shift;  // of a tile's query rows
  int* err;
  __device__ __forceinline__ int rows_per_tile() const { return 1 << row_shift; }
};
// Sizes of tiles are powers of two, and shifts: a CTA runs the search for its run once, and fetches every instruction of a division
// for it.
constexpr int KEY_SHIFT = 6, KEYS_PER_TILE = 1 << KEY_SHIFT;

// One tree: sizes in units.
struct Tree {
  int first, n, ctx;      // first row, nodes (-1: not inside the rows), stored tokens
  int lo_tile, key_tiles; // first key tile any node sees, key tiles from there
  int row_tiles;
};

__device__ __forceinline__ Tree load_tree(const Shape& sh, int s) {
  Tree t;
  const int end = sh.node_start[s + 1];
  t.first = sh.node_start[s];
  t.n = t.first >= 0 && end >= t.first && end <= sh.rows ? end - t.first : -1;
  t.ctx = min(max(0, sh.ctx_len[s]), sh.most_ctx);
  // the root sees furthest back: keys from ctx - window + 1
  const int lo = sh.window > 0 ? max(0, t.ctx - sh.window + 1) : 0;
  t.lo_tile = lo >> KEY_SHIFT;
  t.key_tiles = t.n > 0 ? ((t.ctx + t.n + KEYS_PER_TILE - 1) >> KEY_SHIFT) - t.lo_tile : 0;
  t.row_tiles = (max(t.n, 0) * sh.G + sh.rows_per_tile() - 1) >> sh.row_shift;
  return t;
}
// Units of a tree in one of its row tiles.
__device__ __forceinline__ int units_of(const Shape& sh, const Tree& t) { return t.key_tiles * sh.KVH; }

__device__ __forceinline__ int warp_sum_int(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int warp_scan(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// How the units are cut into runs, one per CTA.
struct Cut {
  int total, chunk;   // all units; units of a run (at least min_units)
  int of_first;       // units of the first row tile
  int per_row_tile;   // > 0: so many CTAs for each row tile, whose runs begin and end with it
  __device__ __forceinline__ int begin(int cta) const {
    if (per_row_tile == 0) return (int)min((long)chunk * cta, (long)total);
    const int tile = cta / per_row_tile;
    return min(tile * of_first + (cta - tile * per_row_tile) * chunk, (tile + 1) * of_first);
  }
  __device__ __forceinline__ int end(int cta) const {
    if (per_row_tile == 0) return (int)min((long)chunk * (cta + 1), (long)total);
    const int tile = cta / per_row_tile;
    return min(tile * of_first + (cta - tile * per_row_tile + 1) * chunk, (tile + 1) * of_first);
  }
  __device__ __forceinline__ int owner(int u) const {
    if (per_row_tile == 0) return u / chunk;
    const int tile = u / of_first;
    return tile * per_row_tile + (u - tile * of_first) / chunk;
  }
};
// Where a CTA's run begins.
struct Found {
  Cut cut;
  int cta;                  // whose run it is
  int seq, row_tile, start; // the tree (-1: the run is empty), the row tile, first unit of that tree in that row tile
  Tree tree;
};
// Called by whole warps.  The trees of up to 32 requests are read once.  Block b has the run of CTA b; with runs per row tile, the
// blocks take the row tiles in turn, so that where there are fewer units than CTAs the blocks with one lie on as many SMs.
__device__ __forceinline__ Found find_run(const Shape& sh, int block, int ctas) {
  constexpr int HELD = 1;
  const int lane = threadIdx.x & 31;
  Found f = {};
  f.cta = block;
  f.seq = -1;
  Tree held[HELD];
  int all = 0, of_first = 0, most = 0;
  bool outside = false;
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    held[k] = {};
    if (k * 32 + lane < sh.S) held[k] = load_tree(sh, k * 32 + lane);
  }
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    all += units_of(sh, held[k]) * held[k].row_tiles;
    of_first += units_of(sh, held[k]);
    most = max(most, held[k].row_tiles);
    outside |= held[k].n < 0;
  }
#pragma unroll 1
  for (int s = HELD * 32 + lane; s < sh.S; s += 32) {
    const Tree t = load_tree(sh, s);
    all += units_of(sh, t) * t.row_tiles;
    of_first += units_of(sh, t);
    most = max(most, t.row_tiles);
    outside |= t.n < 0;
  }
  if (outside) atomicOr(sh.err, DSP_ERR_BAD_TREE);
  Cut& cut = f.cut;
  cut.total = warp_sum_int(all);
  if (cut.total == 0) return f;
  cut.of_first = warp_sum_int(of_first);
  // the same number of row tiles in all trees (no tree has more, and their units add up to it): each gets as many CTAs
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  cut.per_row_tile = most > 1 && most <= ctas && (long)most * cut.of_first == cut.total ? ctas / most : 0;
  cut.chunk = cut.per_row_tile > 0 ? (cut.of_first + cut.per_row_tile - 1) / cut.per_row_tile : (cut.total + ctas - 1) / ctas;
  cut.chunk = max(cut.chunk, sh.min_units);
  if (cut.per_row_tile > 0) {
    if (block >= cut.per_row_tile * most) return f;
    f.cta = block % most * cut.per_row_tile + block / most;
  }
  const int cta = f.cta;
  const int u = cut.begin(cta);
  if (u >= cut.end(cta)) return f;
  // of lane's tree of the k-th 32 in a row tile
  auto units = [&](const Tree& t, int tile) -> int { return t.row_tiles > tile ? units_of(sh, t) : 0; };
  int before = 0;
#pragma unroll 1
  for (int tile = 0;; ++tile) {
    int of_tile = 0;
#pragma unroll
    for (int k = 0; k < HELD; ++k) of_tile += units(held[k], tile);
#pragma unroll 1
    for (int s = HELD * 32 + lane; s < sh.S; s += 32) of_tile += units(load_tree(sh, s), tile);
    of_tile = warp_sum_int(of_tile);
    if (u >= before + of_tile) {
      before += of_tile;
      continue;  // (ends: u is below the total)
    }
    auto look = [&](const Tree& t, int s0) -> bool {
      const int n = units(t, tile);
      const int upto = before + warp_scan(n);
      const uint32_t past = __ballot_sync(0xffffffffu, upto > u);
      if (past == 0u) {
        before = __shfl_sync(0xffffffffu, upto, 31);
        return false;
      }
      const int who = __ffs(past) - 1;
      f.seq = s0 + who;
      f.row_tile = tile;
      f.start = __shfl_sync(0xffffffffu, upto - n, who);
      f.tree.first = __shfl_sync(0xffffffffu, t.first, who);
      f.tree.n = __shfl_sync(0xffffffffu, t.n, who);
      f.tree.ctx = __shfl_sync(0xffffffffu, t.ctx, who);
      f.tree.lo_tile = __shfl_sync(0xffffffffu, t.lo_tile, who);
      f.tree.key_tiles = __shfl_sync(0xffffffffu, t.key_tiles, who);
      f.tree.row_tiles = __shfl_sync(0xffffffffu, t.row_tiles, who);
      return true;
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (look(held[k], k * 32)) return f;
#pragma unroll 1
    for (int s0 = HELD * 32; s0 < sh.S; s0 += 32) {
      Tree t = {};
      if (s0 + lane < sh.S) t = load_tree(sh, s0 + lane);
      if (look(t, s0)) return f;
    }
    return f;
  }
}

// One item's part of a CTA's run.
struct Share {
  int seq, first, n, ctx;  // the tree (seq -1: the run has ended)
  int head, row_tile;
  int kt_begin, kt_end;    // key tiles, counted from key 0
  int slot;                // scratch slot of the partial result, -1: the item is finished here
};

// The item that begins in a CTA and ends in a later one, for the kernel that merges its partial results: written by that CTA.
struct Split {
  int parts;                  // CTAs that have a part (0: there is no such item)
  int first, row0, rows, head;
  int unused[3];
};

// A CTA's walk over its run of units, one item's share at a time.
struct Walk {
  int cta;
  int u, end;
  Cut cut;
  int item_start, key_tiles, lo_tile;
  Share at;

  // Called by whole warps.  False: this CTA has no work.
  __device__ __forceinline__ bool begin(const Shape& sh, int block, int ctas) {
    const Found f = find_run(sh, block, ctas);
    cta = f.cta;
    if (f.seq < 0) return false;
    cut = f.cut;
    u = cut.begin(cta);
    end = cut.end(cta);
    at.seq = f.seq;
    at.row_tile = f.row_tile;
    enter(f.tree);
    at.head = (u - f.start) / key_tiles;
    item_start = f.start + at.head * key_tiles;
    share();
    return true;
  }
  __device__ __forceinline__ void enter(const Tree& t) {
    at.first = t.first;
    at.n = t.n;
    at.ctx = t.ctx;
    key_tiles = t.key_tiles;
    lo_tile = t.lo_tile;
  }
  __device__ __forceinline__ void share() {
    const int item_end = item_start + key_tiles, stop = min(end, item_end);
    at.kt_begin = lo_tile + (u - item_start);
    at.kt_end = at.kt_begin + (stop - u);
    at.slot = u == item_start ? (stop == item_end ? -1 : 2 * cta + 1) : 2 * cta;
  }
  // What the merging kernel has to know of the present share (of the last one of the run, if that is an item's beginning).
  __device__ __forceinline__ Split split(const Shape& sh) const {
    Split x = {};
    if (at.slot == 2 * cta + 1) {
      x.parts = cut.owner(item_start + key_tiles - 1) - cta + 1;
      x.first = at.first;
      x.row0 = at.row_tile << sh.row_shift;
      x.rows = min(sh.rows_per_tile(), at.n * sh.G - x.row0);
      x.head = at.head;
    }
    return x;
  }
  __device__ __forceinline__ bool next(const Shape& sh) {
    u += at.kt_end - at.kt_begin;
    if (u >= end) return false;
    item_start = u;
    if (++at.head == sh.KVH) {
      at.head = 0;
      Tree t;
      do {  // (there is such a tree: units are left)
        if (++at.seq == sh.S) {
          at.seq = 0;
          ++at.row_tile;
        }
        t = load_tree(sh, at.seq);
      } while (t.row_tiles <= at.row_tile);
      enter(t);
    }
    share();
    return true;
  }
};

}  // namespace tree

// Scratch of a call: part_o [2 ctas][rows_per_tile][D] floats, part_ml [2 ctas][rows_per_tile] pairs (maximum in the base-2
// domain, sum), splits [ctas].
struct TreeScratch {
  float *part_o, *part_ml;
  tree::Split* splits;
};
inline TreeScratch tree_scratch(float* scratch, long ctas, long rows_per_tile, long D) {
  TreeScratch s;
  s.part_o = scratch;
  s.part_ml = s.part_o + 2 * ctas * rows_per_tile * D;
  s.splits = reinterpret_cast<tree::Split*>(s.part_ml + 4 * ctas * rows_per_tile);
  return s;
}

// Merges the partial results of the items that several CTAs share (tree_attn.cu).
cudaError_t tree_combine(const TreeScratch& scratch, void* out, long out_stride, int G, int D, int rows_per_tile, int ctas,
                         int dtype, cudaStream_t stream);

// The attention's arguments, checked.
constexpr int ROW_SHIFT_TENSOR_CORES = 7;  // 128 rows a tile of the tensor-core kernel
struct DspTreeAttention {
  tree::Shape sh;
  const void *q, *k_pool, *v_pool;
  const int *page_table, *depth;
  const unsigned long long* visible;
  void* out;
  TreeScratch scratch;
  long q_stride, out_stride;
  int pt_stride, table_width, words, D, page_size, num_pages, ctas;
  float scale;
  int* err;
};
