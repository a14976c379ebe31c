// How the attention of sequences with a shared beginning is cut among CTAs, shared by its kernels.
//
// Group g has the sequences group_start[g] .. group_start[g + 1] - 1, one query row each (G rows a key/value head).  Its first
// P_g = prefix_len[g] tokens are the same for all of them and are read through the pages of its first sequence.  A segment is
// either such a beginning with the rows of all the group's sequences, or one sequence's keys behind it with its own G rows (a
// group of one has no shared part: all its keys are one segment).  An item is one tile of query rows of one key/value head of
// one segment; it walks the key tiles of 64 that any of its rows sees.  A unit is one key tile of one item.  All units, in the order
// (shared parts, sequences; row tile, head, key tile), are cut into equal runs, one per CTA, wherever that falls, so that few long
// beginnings load every SM as well as many short sequences, and nothing about lengths is needed on the host.
//
// Every item leaves a partial result (32-bit sums that are not divided yet, running maximum, sum of weights): in the place of its
// rows, `rows_o`, where one CTA had all of it, else one in each CTA's scratch slots (2 c + 1 for the item that begins in CTA c,
// 2 c for the one that began before).  A record of each item says which; shared_combine_kernel merges a row's two items.
#pragma once
#include "rows_schedule.cuh"

namespace shared {

constexpr int MAX_GROUPS = 1024;  // of a call: a CTA holds what it has to know of all of them

struct Shape {
  const int *group_start, *prefix_len, *ctx_len;
  int groups, KVH, G, window, min_units;
  int rows;       // sequences: a group that is not inside them is recorded and left out
  int most_ctx;   // tokens that a sequence's pages hold
  int row_shift;  // of a tile's query rows
  int* err;
  __host__ __device__ __forceinline__ int rows_per_tile() const { return 1 << row_shift; }
  // items are numbered by row tiles: those of shared parts by their group's first row, then those of sequences
  __host__ __device__ __forceinline__ long shared_tiles() const { return ((long)rows * G >> row_shift) + groups + 1; }
  __host__ __device__ __forceinline__ int tiles_of_sequence() const { return (G + rows_per_tile() - 1) >> row_shift; }
  __host__ __device__ __forceinline__ long items() const { return (shared_tiles() + (long)rows * tiles_of_sequence()) * KVH; }
  __device__ __forceinline__ long item(int part, int group, int first, int row_tile, int head) const {
    const long tile = part == 0 ? ((long)first * G >> row_shift) + group + row_tile
                                : shared_tiles() + (long)first * tiles_of_sequence() + row_tile;
    return tile * KVH + head;
  }
  __device__ __forceinline__ int length(int row) const { return min(max(0, ctx_len[row]), most_ctx); }
};

// The group of a row, -1: in none.
__device__ __forceinline__ int group_of(const int* start, int groups, int rows, int row) {
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return start[lo] <= row && row < start[lo + 1] && start[lo] >= 0 && start[lo + 1] <= rows ? lo : -1;
}

// What a CTA has to know of the groups, in shared memory, and where its run begins.
struct Plan {
  int start[MAX_GROUPS + 1], prefix[MAX_GROUPS], shortest[MAX_GROUPS], longest[MAX_GROUPS];
  int of_warp[32];
  int total, chunk;               // all units; units of a run
  int segment, segment_start;     // of the CTA's first unit
};

struct Segment {
  int seq, group, part, first, n;  // sequence whose pages are read; first row and number of rows
  int from, begin, end;            // first key of the segment; the keys that any of its rows sees
  int all_begin, all_end;          // the keys that all of them see
  int lo_tile, key_tiles, row_tiles;
};

__device__ __forceinline__ Segment segment(const Shape& sh, const Plan& plan, int s) {
  Segment x = {};
  const int row = s - sh.groups;
  if (row < 0) {
    x.group = s;
    x.part = 0;
    x.first = plan.start[s];
    x.n = plan.start[s + 1] - x.first;
    if (x.first < 0 || plan.start[s + 1] > sh.rows || x.n < 2) return x;
    x.end = min(plan.prefix[s], plan.longest[s]);
    x.all_end = min(plan.prefix[s], plan.shortest[s]);
    if (sh.window > 0) {
      x.begin = max(0, plan.shortest[s] - sh.window);
      x.all_begin = max(0, plan.longest[s] - sh.window);
    }
  } else {
    x.group = group_of(plan.start, sh.groups, sh.rows, row);
    x.part = 1;
    x.first = row;
    x.n = 1;
    if (x.group < 0) return x;
    const int length = sh.length(row);
    x.from = plan.start[x.group + 1] - plan.start[x.group] > 1 ? plan.prefix[x.group] : 0;
    x.begin = x.all_begin = max(x.from, sh.window > 0 ? length - sh.window : 0);
    x.end = x.all_end = length;
  }
  x.seq = x.first;
  x.lo_tile = x.begin >> KEY_SHIFT;
  x.key_tiles = x.end > x.begin ? ((x.end + KEYS_PER_TILE - 1) >> KEY_SHIFT) - x.lo_tile : 0;
  x.row_tiles = (x.n * sh.G + sh.rows_per_tile() - 1) >> sh.row_shift;
  return x;
}
__device__ __forceinline__ int units_of(const Shape& sh, const Segment& x) { return x.key_tiles * x.row_tiles * sh.KVH; }

// By the whole block.
__device__ __forceinline__ void make_plan(const Shape& sh, Plan& plan, int cta, int ctas) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  for (int g = tid; g <= sh.groups; g += threads) {
    plan.start[g] = sh.group_start[g];
    if (g == sh.groups) break;
    plan.prefix[g] = min(max(0, sh.prefix_len[g]), sh.most_ctx);
    plan.shortest[g] = 0x7fffffff;
    plan.longest[g] = 0;
  }
  if (tid == 0) plan.segment = -1;
  __syncthreads();
  for (int g = tid; g < sh.groups; g += threads)
    if (plan.start[g] < 0 || plan.start[g + 1] < plan.start[g] || plan.start[g + 1] > sh.rows) atomicOr(sh.err, DSP_ERR_BAD_GROUP);
  for (int row = tid; row < sh.rows; row += threads) {
    const int length = sh.length(row), g = group_of(plan.start, sh.groups, sh.rows, row);
    if (g < 0) continue;
    atomicMin(&plan.shortest[g], length);
    atomicMax(&plan.longest[g], length);
  }
  __syncthreads();
  // a thread has neighbouring segments
  const int segments = sh.groups + sh.rows, each = (segments + threads - 1) / threads;
  const int s0 = min(tid * each, segments), s1 = min(s0 + each, segments);
  int mine = 0;
  for (int s = s0; s < s1; ++s) mine += units_of(sh, segment(sh, plan, s));
  int upto = warp_scan(mine);
  if (lane == 31) plan.of_warp[warp] = upto;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < threads >> 5; ++w) {
    if (w < warp) upto += plan.of_warp[w];
    total += plan.of_warp[w];
  }
  const int chunk = max((total + ctas - 1) / ctas, sh.min_units);
  const long u = (long)chunk * cta;
  if (u < total && u < upto && u >= upto - mine) {
    int at = upto - mine;
    for (int s = s0; s < s1; ++s) {
      const int n = units_of(sh, segment(sh, plan, s));
      if (u < at + n) {
        plan.segment = s;
        plan.segment_start = at;
        break;
      }
      at += n;
    }
  }
  if (tid == 0) {
    plan.total = total;
    plan.chunk = chunk;
  }
  __syncthreads();
}

// One item's part of a CTA's run.
struct Share {
  int seq;                 // whose pages are read (-1: the run has ended)
  int part, group, first, n;
  int from, begin, end, all_begin, all_end;
  int head, row_tile;
  int kt_begin, kt_end;    // key tiles, counted from key 0
  int slot;                // scratch slot of the partial result, -1: in the place of its rows
};

// Where an item's partial results are: in `parts` CTAs from `cta` on (one: in the place of its rows).
struct Record {
  int cta, parts;
};
struct Note {
  long item;  // -1: the share does not begin its item
  Record record;
};

// A CTA's walk over its run of units, one item's share at a time.
struct Walk {
  int cta;
  int u, end, chunk, segment_at;
  int item_start, key_tiles, lo_tile, row_tiles;
  Share at;

  __device__ __forceinline__ bool begin(const Shape& sh, const Plan& plan, int block, int) {
    cta = block;
    at.seq = -1;
    if (plan.segment < 0) return false;
    chunk = plan.chunk;
    u = chunk * cta;
    end = (int)min((long)u + chunk, (long)plan.total);
    segment_at = plan.segment;
    enter(segment(sh, plan, segment_at));
    const int item = (u - plan.segment_start) / key_tiles;
    item_start = plan.segment_start + item * key_tiles;
    at.row_tile = item / sh.KVH;
    at.head = item - at.row_tile * sh.KVH;
    share();
    return true;
  }
  __device__ __forceinline__ void enter(const Segment& x) {
    at.seq = x.seq;
    at.part = x.part;
    at.group = x.group;
    at.first = x.first;
    at.n = x.n;
    at.from = x.from;
    at.begin = x.begin;
    at.end = x.end;
    at.all_begin = x.all_begin;
    at.all_end = x.all_end;
    key_tiles = x.key_tiles;
    lo_tile = x.lo_tile;
    row_tiles = x.row_tiles;
  }
  __device__ __forceinline__ void share() {
    const int item_end = item_start + key_tiles, stop = min(end, item_end);
    at.kt_begin = lo_tile + (u - item_start);
    at.kt_end = at.kt_begin + (stop - u);
    at.slot = u == item_start ? (stop == item_end ? -1 : 2 * cta + 1) : 2 * cta;
  }
  __device__ __forceinline__ Note split(const Shape& sh) const {
    Note x = {-1, {cta, 1}};
    if (u == item_start) {
      x.item = sh.item(at.part, at.group, at.first, at.row_tile, at.head);
      x.record.parts = (item_start + key_tiles - 1) / chunk - cta + 1;
    }
    return x;
  }
  __device__ __forceinline__ bool next(const Shape& sh, const Plan& plan) {
    u += at.kt_end - at.kt_begin;
    if (u >= end) return false;
    item_start = u;
    if (++at.head == sh.KVH) {
      at.head = 0;
      if (++at.row_tile == row_tiles) {
        at.row_tile = 0;
        Segment x;
        do {  // (there is such a segment: units are left)
          x = segment(sh, plan, ++segment_at);
        } while (x.key_tiles == 0);
        enter(x);
      }
    }
    share();
    return true;
  }
};

}  // namespace shared

// Scratch of a call: part_o [2 ctas][rows of a tile][D] floats, part_ml [2 ctas][rows of a tile] pairs (maximum in the base-2
// domain, sum), rows_o [2][rows H][D], rows_ml [2][rows H] pairs, records [items].
struct SharedScratch {
  float *part_o, *part_ml, *rows_o, *rows_ml;
  shared::Record* records;
};

// The attention's arguments, checked.
struct DspSharedAttention {
  shared::Shape sh;
  const void *q, *k_pool, *v_pool;
  const int* page_table;
  void* out;
  SharedScratch scratch;
  long q_stride, out_stride;
  int pt_stride, table_width, D, page_size, num_pages, ctas;
  float scale;
  int* err;
};

// What the kernels over rows have to know of sequences with a shared beginning: a row sees an interval of keys.
struct SharedWork {
  typedef DspSharedAttention Args;
  typedef shared::Shape Shape;
  typedef shared::Share Share;
  typedef shared::Walk Walk;
  typedef shared::Plan Plan;
  static constexpr bool ROW_PARTS = true;  // items that are finished where they began are partial results all the same
  struct Row {
    int lo, hi;
  };
  static __device__ __forceinline__ void make_plan(const Shape& sh, Plan& plan, int cta, int ctas) { shared::make_plan(sh, plan, cta, ctas); }
  static __device__ __forceinline__ void note(const Args& a, int, const shared::Note& x, bool) {
    if (x.item >= 0) a.scratch.records[x.item] = x.record;
  }
  static __device__ __forceinline__ void note_none(const Args&, int) {}
  static __device__ __forceinline__ int key_begin(const Shape&, const Share& t) { return t.begin; }
  static __device__ __forceinline__ int key_end(const Share& t) { return t.end; }
  static __device__ __forceinline__ bool whole(const Shape&, const Share& t, int key0) {
    return key0 >= t.all_begin && key0 + KEYS_PER_TILE <= t.all_end;
  }
  static __device__ __forceinline__ Row row(const Args& a, const Share& t, int node) {
    const int length = a.sh.length(node);
    return {max(t.from, a.sh.window > 0 ? length - a.sh.window : 0), min(t.end, length)};
  }
  static __device__ __forceinline__ bool any_hidden(const Shape&, const Share&, const Row& row, int key0) {
    return __any_sync(0xffffffffu, key0 < row.lo || key0 + KEYS_PER_TILE > row.hi);
  }
  static __device__ __forceinline__ unsigned long long seen_keys(const Args&, const Share&, const Row& row, int key0) {
    const int lo = max(row.lo - key0, 0), n = min(row.hi - key0, KEYS_PER_TILE) - lo;  // bits lo .. lo + n - 1
    return n <= 0 ? 0ull : n >= 64 ? ~0ull : ((1ull << n) - 1ull) << lo;
  }
  static __device__ __forceinline__ bool sees(const Args&, const Share&, const Row& row, int key) { return key >= row.lo && key < row.hi; }
  // place of a tile's row rr (counted from the segment's first) in rows_o and rows_ml
  static __device__ __forceinline__ size_t row_part(const Shape& sh, const Share& t, int rr) {
    const int node = rr / sh.G;
    return ((size_t)t.part * sh.rows + t.first + node) * sh.KVH * sh.G + t.head * sh.G + (rr - node * sh.G);
  }
};
