// How the attention of sequences with a shared beginning is cut among CTAs, shared by its kernels.
//
// Group g has the sequences group_start[g] .. group_start[g + 1] - 1, one query row each (G rows a key/value head).  Its first
// P_g = prefix_len[g] tokens are the same for all of them and are read through the pages of its first sequence.  A segment is
// either such a beginning with the rows of all the group's sequences, or one sequence's keys behind it with its own G rows (a
// group of one has no shared part: all its keys are one segment).  An item is one tile of query rows of one key/value head of
// one segment; it walks the key tiles of 64 that any of its rows sees, and is counted as so many units and `extra` more, which stand for
// its beginning and end, all twice where a tile has more than `heavy` rows.  All units, in the order (shared parts, sequences; row tile,
// head, key tile), are cut into equal runs, one per CTA, wherever that falls, so that few long beginnings load every SM as well as many
// short sequences, and nothing about lengths is needed on the host.
//
// Two kernels may share the work: beginnings with more than `many` rows a head go to one whose tiles have 256 rows, the rest to
// one with smaller tiles.  Where all beginnings of the first have R row tiles, teams of R CTAs walk the same keys with one row
// tile each, which then come from memory once and from the L2 for the others.  CTAs beyond the last whole team have nothing to do
// (75 row tiles, some 2,400 sequences of 8 rows a head, leave 73 of 148 idle), and a last row tile of few rows has as many as a full one.
//
// Every item leaves a partial result (32-bit sums that are not divided yet, running maximum, sum of weights): in the place of its
// rows, `rows_o`, where one CTA had all of it, else one in each CTA's scratch slots (2 c + 1 for the item that begins in CTA c,
// 2 c for the one that began before).  A record of each item says which; shared_combine_kernel merges a row's two items.
//
// Which groups there are is settled before anything is counted: one that is not inside the rows, or does not begin behind those before
// it, is left out, so that the groups that are there ascend and a row is in one of them at most.  All that counts units, walks them or
// merges goes by that (a row that lay in two groups for one of them made runs longer than what there was to walk).
#pragma once
#include "rows_schedule.cuh"

namespace shared {

constexpr int MAX_GROUPS = 1024;  // of a call: a CTA holds what it has to know of all of them while it finds its run

struct Shape {
  const int *group_start, *prefix_len, *ctx_len;
  int groups, KVH, G, window, min_units, extra;
  int rows;       // sequences: a group that is not inside them is recorded and left out
  int most_ctx;   // tokens that a sequence's pages hold
  int row_shift;  // of a tile's query rows
  int heavy;      // a row tile of more rows takes two units a key tile
  int many;       // shared parts of more rows a head are for the kernel of many rows
  int is_many;    // that kernel's shape
  int* err;
  __host__ __device__ __forceinline__ int rows_per_tile() const { return 1 << row_shift; }
  // items are numbered by row tiles: those of shared parts by their group's first row, then those of sequences
  __host__ __device__ __forceinline__ long shared_tiles() const { return ((long)rows * G >> row_shift) + groups + 1; }
  __host__ __device__ __forceinline__ int tiles_of_sequence() const { return (G + rows_per_tile() - 1) >> row_shift; }
  __host__ __device__ __forceinline__ long items() const {
    return (shared_tiles() + (is_many ? 0 : (long)rows * tiles_of_sequence())) * KVH;
  }
  __device__ __forceinline__ long item(int part, int group, int first, int row_tile, int head) const {
    const long tile = part == 0 ? ((long)first * G >> row_shift) + group + row_tile
                                : shared_tiles() + (long)first * tiles_of_sequence() + row_tile;
    return tile * KVH + head;
  }
  __device__ __forceinline__ int length(int row) const { return min(max(0, ctx_len[row]), most_ctx); }
};

// Where groups begin, in shared memory.
struct Starts {
  int start[MAX_GROUPS + 1];
  uint32_t out[MAX_GROUPS / 32];  // bit g % 32 of word g / 32: group g is left out

  struct Own {  // begin and end of the group with the thread's number
    int first, end;
  };
  static __device__ __forceinline__ Own ask(const Shape& sh) {
    const int tid = threadIdx.x;
    return tid < sh.groups ? Own{sh.group_start[tid], sh.group_start[tid + 1]} : Own{0, 0};
  }
  // By the whole block, which meets: brings them (`own`: asked for before, with what else is wanted, so that the answers come together).
  // Returns whether some are left out; then the others' places stay as they are, and what is left out fills the gaps between them.
  __device__ __forceinline__ bool bring(const Shape& sh, const Own& own) {
    const int tid = threadIdx.x;
    bool bad = false;
    for (int g = tid; g < sh.groups; g += blockDim.x) {
      const int first = g == tid ? own.first : sh.group_start[g], end = g == tid ? own.end : sh.group_start[g + 1];
      start[g] = first;
      if (g + 1 == sh.groups) start[g + 1] = end;
      bad |= first < 0 || end < first || end > sh.rows;
    }
    if (tid < MAX_GROUPS / 32) out[tid] = 0;
    if (!__syncthreads_or(bad)) return false;
    if (tid == 0) {
      int at = 0, end = start[0];  // of the last group that is there; in the list as it came
      for (int g = 0; g < sh.groups; ++g) {
        const int first = end;
        end = start[g + 1];
        const bool there = first >= at && end >= first && end <= sh.rows;
        start[g] = there ? first : at;
        if (there)
          at = end;
        else
          out[g >> 5] |= 1u << (g & 31);
      }
      start[sh.groups] = at;
    }
    __syncthreads();
    return true;
  }
  __device__ __forceinline__ bool left_out(int g) const { return (out[g >> 5] >> (g & 31)) & 1u; }
};
// The group of a row, -1: in none.  The starts ascend.
__device__ __forceinline__ int group_of(const int* start, int groups, int row) {
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return start[lo] <= row && row < start[lo + 1] ? lo : -1;
}
__device__ __forceinline__ int group_of(const Starts& s, int groups, int row) {
  const int g = group_of(s.start, groups, row);
  return g >= 0 && !s.left_out(g) ? g : -1;
}

// What a CTA has to know of the groups while it finds its run.
struct Groups {
  Starts starts;
  int prefix[MAX_GROUPS], shortest[MAX_GROUPS], longest[MAX_GROUPS];
  int of_warp[32], most_tiles[32], least_tiles[32];
};
struct Segment {
  int group, part, first, n;   // first row and number of rows; the first one's pages are read
  int from, begin, end;        // first key of the segment; the keys that any of its rows sees
  int all_begin, all_end;      // the keys that all of them see
  int lo_tile, key_tiles, row_tiles;
  int weight, last_weight;     // units a key tile of a whole row tile, and of the last one
};

__device__ __forceinline__ void set_weights(const Shape& sh, Segment& x) {
  x.weight = sh.rows_per_tile() > sh.heavy ? 2 : 1;
  x.last_weight = x.n * sh.G - ((x.row_tiles - 1) << sh.row_shift) > sh.heavy ? 2 : 1;
}
// The shared part of group g (`first` -1: it is left out), whose sequences have between `shortest` and `longest` tokens.
__device__ __forceinline__ Segment shared_part(const Shape& sh, int g, int first, int end, int prefix, int shortest, int longest) {
  Segment x = {};
  x.group = g;
  x.first = first;
  x.n = end - first;
  if (first < 0 || x.n < 2 || ((long)x.n * sh.G > sh.many) != (sh.is_many != 0)) return x;
  x.end = min(prefix, longest);
  x.all_end = min(prefix, shortest);
  if (sh.window > 0) {
    x.begin = max(0, shortest - sh.window);
    x.all_begin = max(0, longest - sh.window);
  }
  x.lo_tile = x.begin >> KEY_SHIFT;
  x.key_tiles = x.end > x.begin ? ((x.end + KEYS_PER_TILE - 1) >> KEY_SHIFT) - x.lo_tile : 0;
  x.row_tiles = (x.n * sh.G + sh.rows_per_tile() - 1) >> sh.row_shift;
  set_weights(sh, x);
  return x;
}
// The own part of a row of group g (first .. end - 1), -1: of none.
__device__ __forceinline__ Segment own_part(const Shape& sh, int row, int g, int first, int end, int prefix) {
  Segment x = {};
  x.group = g;
  x.part = 1;
  x.first = row;
  x.n = 1;
  if (g < 0 || sh.is_many) return x;
  const int length = sh.length(row);
  x.from = end - first > 1 ? prefix : 0;
  x.begin = x.all_begin = max(x.from, sh.window > 0 ? length - sh.window : 0);
  x.end = x.all_end = length;
  x.lo_tile = x.begin >> KEY_SHIFT;
  x.key_tiles = x.end > x.begin ? ((x.end + KEYS_PER_TILE - 1) >> KEY_SHIFT) - x.lo_tile : 0;
  x.row_tiles = sh.tiles_of_sequence();
  set_weights(sh, x);
  return x;
}
// `near`: a group that is there and that the row may be in, looked at first.
__device__ __forceinline__ Segment segment(const Shape& sh, const Groups& groups, int s, int near = -1) {
  const int row = s - sh.groups;
  const int* start = groups.starts.start;
  if (row < 0)
    return shared_part(sh, s, groups.starts.left_out(s) ? -1 : start[s], start[s + 1], groups.prefix[s], groups.shortest[s], groups.longest[s]);
  if (near < 0 || row < start[near] || row >= start[near + 1]) near = group_of(groups.starts, sh.groups, row);
  const int at = max(near, 0);
  return own_part(sh, row, near, start[at], start[at + 1], groups.prefix[at]);
}
// Units of a segment, or with teams of one of its row tiles (which all weigh the same then).
__device__ __forceinline__ int units_of(const Shape& sh, const Segment& x, bool teams) {
  if (x.key_tiles <= 0) return 0;
  return sh.KVH * (x.key_tiles + sh.extra) * (teams ? 1 : (x.row_tiles - 1) * x.weight + x.last_weight);
}

// Where a CTA's run begins.
constexpr int AHEAD = 24;  // segments from there on that are worked out while all groups are at hand
struct Run {
  int total, chunk;            // all units (of one row tile, with teams); units of a run
  int teams;                   // CTAs that walk the same keys
  int segment, segment_start;  // of the CTA's first unit (-1: there is none)
  int segments;
  bool some_out;               // groups are left out, these:
  uint32_t out[MAX_GROUPS / 32];
  Segment ahead[AHEAD];
};
struct Plan {
  Groups groups;
  Run run;
};

// By the whole block.
__device__ __forceinline__ void make_plan(const Shape& sh, Groups& groups, Run& run, int cta, int ctas) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int own_length = tid < sh.rows ? sh.length(tid) : 0;  // (asked for with the groups)
  const int own_prefix = tid < sh.groups ? sh.prefix_len[tid] : 0;
  const Starts::Own own_group = Starts::ask(sh);
  for (int g = tid; g < sh.groups; g += threads) {
    groups.prefix[g] = min(max(0, g == tid ? own_prefix : sh.prefix_len[g]), sh.most_ctx);
    groups.shortest[g] = 0x7fffffff;
    groups.longest[g] = 0;
  }
  if (tid == 0) run.segment = -1;
  const bool some_out = groups.starts.bring(sh, own_group);
  if (some_out) {
    if (tid == 0) atomicOr(sh.err, DSP_ERR_BAD_GROUP);
    if (tid < MAX_GROUPS / 32) run.out[tid] = groups.starts.out[tid];
  }
  for (int row = tid; row < sh.rows; row += threads) {
    const int length = row == tid ? own_length : sh.length(row), g = group_of(groups.starts, sh.groups, row);
    if (g < 0) continue;
    atomicMin(&groups.shortest[g], length);
    atomicMax(&groups.longest[g], length);
  }
  __syncthreads();
  // a thread has neighbouring segments
  const int segments = sh.groups + (sh.is_many ? 0 : sh.rows), each = (segments + threads - 1) / threads;
  const int s0 = min(tid * each, segments), s1 = min(s0 + each, segments);
  int mine = 0, of_first = 0, most = 0, least = 0x7fffffff, near = -1;
  Segment x = {};
  for (int s = s0; s < s1; ++s) {
    x = segment(sh, groups, s, near);
    near = x.part ? x.group : -1;
    mine += units_of(sh, x, false);
    of_first += units_of(sh, x, true);
    if (x.key_tiles > 0) {
      most = max(most, x.row_tiles);
      least = min(least, x.row_tiles);
    }
  }
  bool teams = false;
  if (sh.is_many) {
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) {
      groups.most_tiles[warp] = most;
      groups.least_tiles[warp] = least;
    }
    __syncthreads();
    for (int w = 0; w < threads >> 5; ++w) {
      most = max(most, groups.most_tiles[w]);
      least = min(least, groups.least_tiles[w]);
    }
    teams = most == least && most > 1 && most <= ctas;
  }
  const int team_size = teams ? most : 1;
  if (teams) mine = of_first;
  int upto = warp_scan(mine);
  if (lane == 31) groups.of_warp[warp] = upto;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < threads >> 5; ++w) {
    if (w < warp) upto += groups.of_warp[w];
    total += groups.of_warp[w];
  }
  const int runs = ctas / team_size, chunk = max((total + runs - 1) / runs, sh.min_units);
  const long u = (long)chunk * (cta / team_size);
  if (cta / team_size < runs && u < total && u < upto && u >= upto - mine) {
    int at = upto - mine;
    for (int s = s0; s < s1; ++s) {
      if (each > 1) x = segment(sh, groups, s, near);
      const int n = units_of(sh, x, teams);
      if (u < at + n) {
        run.segment = s;
        run.segment_start = at;
        break;
      }
      at += n;
    }
  }
  if (tid == 0) {
    run.total = total;
    run.chunk = chunk;
    run.teams = team_size;
    run.segments = segments;
    run.some_out = some_out;
  }
  __syncthreads();
  if (run.segment >= 0) {
    if (each == 1) {  // (a thread still has its segment)
      if (tid >= run.segment && tid < min(run.segment + AHEAD, segments)) run.ahead[tid - run.segment] = x;
    } else if (tid < AHEAD && run.segment + tid < segments) {
      run.ahead[tid] = segment(sh, groups, run.segment + tid);
    }
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

// Where an item's partial results are: in `parts` CTAs, cta, cta + stride, ... (one: in the place of its rows).
struct Record {
  int cta;
  short parts, stride;
};
struct Note {
  long item;  // -1: the share does not begin its item
  Record record;
};

// A CTA's walk over its run of units, one item's share at a time.  Called by whole warps.
struct Walk {
  int cta, teams;
  int u, end, chunk, segment_at;
  int item_start, key_tiles, lo_tile, row_tiles;
  int weights[2];          // units a key tile of a whole row tile, and of the last one
  bool begins;             // the share has its item's first key tile
  const Run* run_;
  Share at;

  __device__ __forceinline__ bool begin(const Shape& sh, const Run& run, int block) {
    cta = block;
    run_ = &run;
    at.seq = -1;
    if (run.segment < 0) return false;
    teams = run.teams;
    chunk = run.chunk;
    u = chunk * (cta / teams);
    end = (int)min((long)u + chunk, (long)run.total);
    segment_at = run.segment;
    enter(sh);
    at.row_tile = 0;
    item_start = run.segment_start;
    if (teams > 1) {
      at.row_tile = cta % teams;
    } else {
      const int whole = sh.KVH * (key_tiles + sh.extra) * weights[0];
      at.row_tile = min((u - item_start) / whole, row_tiles - 1);
      item_start += at.row_tile * whole;
    }
    const int cost = (key_tiles + sh.extra) * weight();
    at.head = (u - item_start) / cost;
    item_start += at.head * cost;
    return share(sh) || next(sh);
  }
  __device__ __forceinline__ int weight() const { return teams > 1 ? 1 : at.row_tile + 1 < row_tiles ? weights[0] : weights[1]; }
  // what has to be known of segment `segment_at`; false: it has no keys
  __device__ __forceinline__ bool enter(const Shape& sh) {
    Segment x;
    const int row = segment_at - sh.groups;
    if (segment_at - run_->segment < AHEAD) {
      x = run_->ahead[segment_at - run_->segment];
    } else if (row < 0) {
      const int g = segment_at;
      const bool out = run_->some_out && ((run_->out[g >> 5] >> (g & 31)) & 1u);
      const int first = out ? -1 : sh.group_start[g], last = sh.group_start[g + 1];
      int shortest = 0x7fffffff, longest = 0;
      if (!out)
        for (int r = first + (int)(threadIdx.x & 31); r < last; r += 32) {
          const int length = sh.length(r);
          shortest = min(shortest, length);
          longest = max(longest, length);
        }
      x = shared_part(sh, g, first, last, min(max(0, sh.prefix_len[g]), sh.most_ctx), __reduce_min_sync(0xffffffffu, shortest),
                      __reduce_max_sync(0xffffffffu, longest));
    } else {
      int g = -1;
      if (!run_->some_out) {
        g = group_of(sh.group_start, sh.groups, row);
      } else {  // (the list does not ascend)
        for (int k = threadIdx.x & 31; k < sh.groups; k += 32)
          if (!((run_->out[k >> 5] >> (k & 31)) & 1u) && sh.group_start[k] <= row && row < sh.group_start[k + 1]) g = k;
        g = __reduce_max_sync(0xffffffffu, g);
      }
      const int at = max(g, 0);
      x = own_part(sh, row, g, sh.group_start[at], sh.group_start[at + 1], min(max(0, sh.prefix_len[at]), sh.most_ctx));
    }
    at.seq = at.first = x.first;
    at.part = x.part;
    at.group = x.group;
    at.n = x.n;
    at.from = x.from;
    at.begin = x.begin;
    at.end = x.end;
    at.all_begin = x.all_begin;
    at.all_end = x.all_end;
    key_tiles = x.key_tiles;
    lo_tile = x.lo_tile;
    row_tiles = teams > 1 ? 1 : x.row_tiles;
    weights[0] = x.weight;
    weights[1] = x.last_weight;
    return key_tiles > 0;
  }
  // the run's part of the present item; false: it has no key tile
  __device__ __forceinline__ bool share(const Shape& sh) {
    // (so many key tiles lie in front of a unit of the item)
    const int w = weight(), first_tile = item_start + sh.extra * w, item_end = first_tile + key_tiles * w, stop = min(end, item_end);
    const int before = max(u - first_tile, 0) >> (w - 1), upto = max(stop - first_tile, 0) >> (w - 1);
    begins = before == 0;
    at.kt_begin = lo_tile + before;
    at.kt_end = lo_tile + upto;
    at.slot = begins ? (stop == item_end ? -1 : 2 * cta + 1) : 2 * cta;
    u = stop;
    return upto > before;
  }
  __device__ __forceinline__ Note split(const Shape& sh) const {
    Note x = {-1, {cta, 1, (short)teams}};
    if (begins) {
      x.item = sh.item(at.part, at.group, at.first, at.row_tile, at.head);
      x.record.parts = (short)((item_start + (sh.extra + key_tiles) * weight() - 1) / chunk - cta / teams + 1);
    }
    return x;
  }
  __device__ __forceinline__ bool next(const Shape& sh) {
    do {
      if (u >= end) return false;
      item_start = u;
      if (++at.head == sh.KVH) {
        at.head = 0;
        if (teams > 1 || ++at.row_tile == row_tiles) {
          if (teams == 1) at.row_tile = 0;
          do {
            if (++segment_at >= run_->segments) return false;  // (units are left, so there is such a segment)
          } while (!enter(sh));
        }
      }
    } while (!share(sh));
    return true;
  }
};

}  // namespace shared

// Scratch of a kernel: part_o [2 ctas][rows of a tile][D] floats, part_ml [2 ctas][rows of a tile] pairs (maximum in the base-2
// domain, sum), records [items]; and of both, for items that were not cut: rows_o [2][rows H][D], rows_ml [2][rows H] pairs.
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
  int beside;  // the kernel for few rows is launched behind the one for many
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
  static __device__ __forceinline__ void make_plan(const Shape& sh, Plan& plan, int cta, int ctas) { shared::make_plan(sh, plan.groups, plan.run, cta, ctas); }
  static __device__ __forceinline__ bool begin(Walk& w, const Shape& sh, const Plan& plan, int block, int) { return w.begin(sh, plan.run, block); }
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
