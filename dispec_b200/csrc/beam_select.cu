// The best continuations of every group of beams.
//
// Row r has logits x_v and a score s_r so far; group g has the rows group_start[g] .. group_start[g + 1] - 1.  Its candidates are
// (r, v) with
//     key(r, v) = s_r + (x_v - max x) - log sum_v exp(x_v - max x)
// in 64 bits, the logarithm rounded to 32 (so that equal rows have equal keys, whatever the order of a sum).  Wanted are the n
// largest keys in descending order, ties to the lowest row, then the lowest v.  NaN counts as -inf; what is -inf is no
// candidate; a row whose score is not finite has none; where infinities are the largest logits, they share the mass.
//
// Within a row the order of keys is that of logits, so the n best of a part of a row can be told before its sum is known.
// One pass over the logits: the rows' pieces of 8,192 are dealt out to the CTAs in runs, and a CTA goes through its run with the
// next two pieces on their way into shared memory (bulk copies, where rows begin on 16 bytes).  Of its part of a row it leaves the
// n best in order; and of every piece each warp leaves the maximum and the sum of exponentials of its 1,024 logits, so that sums do
// not depend on how rows are dealt out.
// What does not exceed the n-th best so far is left alone; what does is put aside, and now and then the list is put in order anew by
// counting.  Of a part's first piece a lower bound of the n-th best, which few others reach, costs no search: of each of the 8 warps
// the ceil(n / 8)-th largest of its lanes' maxima, of these the smallest: at least n logits are as large.  (Of a row of 1,093 bfloat16
// logits, which five warps have among them, so do four of these; with all eight, three of them empty, nothing was bounded: 96 rows 15
// us for 307.)  Where too many reach it
// (many equal logits), the piece's exact bound is bisected.  A block a group then merges the sums of its rows' parts and picks n
// of their lists.
//
// What bounds it: loads where there are many (449 rows of 151,936 logits in 32 bits: 56 us for the pieces' kernel, 4.9 TB/s, 68 with the
// groups'; of 151,935, which do not begin on 16 bytes and are loaded one by one, 113 for 77, in bfloat16 110 for 72, each behind a flushed
// L2), else two launches and, behind each other, a piece's way, its list, the groups' bound and their lists (4 rows of 151,936:
// 12 to 14 us; 40 of 152,064 in bfloat16: 18).  Three CTAs an SM with two pieces of 32 KB each are what shared memory holds; a piece's
// 32 logits a thread stay in registers for both passes over them.
#include "packed2.cuh"
#include "tcgen05_common.cuh"
#include "tensor_checks.cuh"

namespace {
constexpr int THREADS = 256, WARPS = THREADS / 32, EACH = 32, PIECE = THREADS * EACH;
constexpr int MAX_COUNT = 8 * 32;  // each warp vouches for an eighth of the wanted, and has so many lanes
constexpr int CAP = 1024;          // candidates of a group that are put in order by counting
constexpr int ASIDE = 32;          // logits that are put aside before a part's list is put in order (which costs as many steps as it has entries)
constexpr int LIST_CAP = 2 * MAX_COUNT + 2 * ASIDE;
constexpr int SAMPLES = 4 * THREADS;

// Numbers in the order of floats; -inf gives the smallest of those that are numbers.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double unordered(unsigned long long o) {
  return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}
constexpr uint32_t NOTHING = 0x007fffffu;  // ordered(-inf)
constexpr unsigned long long NOTHING64 = 0x000fffffffffffffull;

// The k-th largest (from 0) of the lanes' numbers: they are sorted across the warp.
__device__ __forceinline__ uint32_t warp_kth(uint32_t x, int k) {
  const int lane = threadIdx.x & 31;
  if (k < 4) {  // one after the other is quicker
    for (int i = 0; i < k; ++i) {
      const uint32_t those = __ballot_sync(0xffffffffu, x == __reduce_max_sync(0xffffffffu, x));
      if (lane == __ffs(those) - 1) x = 0;
    }
    return __reduce_max_sync(0xffffffffu, x);
  }
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const uint32_t y = __shfl_xor_sync(0xffffffffu, x, step);
      const bool larger = ((lane & step) == 0) == ((lane & size) == 0);  // this lane keeps the larger one
      x = (x > y) == larger ? x : y;
    }
  return __shfl_sync(0xffffffffu, x, k);
}

__device__ __forceinline__ float ex2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Args {
  const void* logits;
  const float* scores;
  const int* group_start;
  int *parent, *token;
  float* score;
  float2* stats;                // [rows][pieces][WARPS] largest logit and sum of exponentials
  // CTA c's part of row r is number c + r (one behind it is left out where both end together, and has no entries)
  uint32_t* parts;              // [rows + ctas] the row, and how many entries the list has
  unsigned long long* lists;    // [rows + ctas][n]: logit in order and its column's complement
  float2* of_rows;              // [rows] largest logit and logarithm of the sum
  long stride;                  // of a row of logits
  int rows, groups, vocab, pieces, n;
  int run;                      // pieces of a CTA
  int bulk;                     // rows begin and end on 16 bytes
  int* err;
};

// How many of the block's numbers reach a bound, by the whole block.
__device__ __forceinline__ int block_sum(int mine, int* of_warp) {
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = mine;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) all += of_warp[w];
  __syncthreads();
  return all;
}

// Where more logits of a piece reach a bound than can be put in order: the n-th largest by bisection, and where its equals are more
// than wanted, the last column taken.  By the whole block; the n go to list[aside] and on.  (Some 280 us a piece: rows of equal logits,
// such as those masked by a finite number, rows that ascend, and counts from 190 on, which the lanes' maxima bound too loosely for the
// list.  4 rows of 151,936, all but 20 logits at -1e9, or ascending: 305 us for 20; 449 rows, 256 wanted 1,149 us, 128 166, 16 77.)
template <int WIDE>
__device__ __noinline__ void exact_bound(const float* x, uint32_t limit, int n, int first, unsigned long long* list,
                                         int aside, int* found, int* of_warp) {
  const int tid = threadIdx.x;
  uint32_t lo = limit, hi = ordered(INFINITY);  // more than n exceed the limit; the answer is above it
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    int c = 0;
#pragma unroll 1
    for (int k = 0; k < EACH; ++k) c += ordered(x[k]) >= mid && x[k] > -INFINITY;
    if (block_sum(c, of_warp) >= n)
      lo = mid;
    else
      hi = mid - 1;
  }
  int above = 0;
#pragma unroll 1
  for (int k = 0; k < EACH; ++k) above += ordered(x[k]) > lo && x[k] > -INFINITY;
  const int equal = n - block_sum(above, of_warp);  // so many of the equals are taken, by column
  int c0 = 0, c1 = PIECE - 1;                       // the last of their columns, counted from `first`
  while (c0 < c1) {
    const int mid = (c0 + c1) / 2;
    int c = 0;
#pragma unroll 1
    for (int k = 0; k < EACH; ++k) c += ordered(x[k]) == lo && WIDE * (tid + k / WIDE * THREADS) + k % WIDE <= mid;
    if (block_sum(c, of_warp) >= equal)
      c1 = mid;
    else
      c0 = mid + 1;
  }
  if (tid == 0) *found = aside;
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < EACH; ++k) {
    const int column = WIDE * (tid + k / WIDE * THREADS) + k % WIDE;
    const uint32_t o = ordered(x[k]);
    if ((o > lo || (o == lo && column <= c0)) && x[k] > -INFINITY) {
      const int at = atomicAdd(found, 1);
      if (at < LIST_CAP) list[at] = (unsigned long long)o << 32 | ~(uint32_t)(first + column);
    }
  }
  __syncthreads();
}

constexpr int PIECES_CTAS = 3, STAGES = 2;  // CTAs an SM
template <typename T>
__global__ void __launch_bounds__(THREADS, PIECES_CTAS)
beam_pieces_kernel(const Args a) {
  extern __shared__ __align__(128) unsigned char stage_bytes[];  // [STAGES][PIECE] logits
  __shared__ unsigned long long lists[2][LIST_CAP];  // the n best so far in order, what was put aside behind them; and in turn
  __shared__ uint32_t bounds[WARPS];
  __shared__ __align__(8) uint64_t landed[STAGES];
  __shared__ int of_warp[WARPS], found;
  constexpr int WIDE = 16 / sizeof(T);  // logits of a load
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
  if (tid == 0) {
    for (int k = 0; k < STAGES; ++k) tc::mbar_init(&landed[k], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: the next kernel looks at the groups before it waits)
  __syncthreads();
  const int begin = blockIdx.x * a.run, end = min(begin + a.run, a.rows * a.pieces);
  auto ask = [&](int p, int k) {  // by one thread: piece p into stage k
    if (p >= end || !a.bulk) return;
    const int row = p / a.pieces, first = (p - row * a.pieces) * PIECE;
    const uint32_t bytes = (uint32_t)min(PIECE, a.vocab - first) * (uint32_t)sizeof(T);
    tc::mbar_expect_tx(&landed[k], bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     tc::smem_u32(stage_bytes + (size_t)k * PIECE * sizeof(T))),
                 "l"((const T*)a.logits + (size_t)row * a.stride + first), "r"(bytes), "r"(tc::smem_u32(&landed[k]))
                 : "memory");
  };
  if (tid == 0)
    for (int k = 0; k < STAGES; ++k) ask(begin + k, k);
  int row = begin / a.pieces, in_row = begin - row * a.pieces;
  bool fresh = true;  // the first piece of a part
  unsigned long long* list = lists[0];
  uint32_t limit = NOTHING;  // the n-th best so far
  int aside = n;             // entries of the list in front of this piece's
#pragma unroll 1
  for (int turn = 0, p = begin; p < end; ++turn, ++p) {
    const int first = in_row * PIECE, there = a.vocab - first;  // columns from the piece's first on
    // Thread t has the columns first + WIDE (t + 256 k) .. + WIDE - 1, however the row lies in memory: equal rows of equal parts
    // give equal sums.
    float x[EACH];
    bool ok = true;
    if (a.bulk) {
      ok = tc::mbar_wait(&landed[turn % STAGES], (turn / STAGES) & 1);
      const uint4* src = reinterpret_cast<const uint4*>(stage_bytes + (size_t)(turn % STAGES) * PIECE * sizeof(T)) + tid;
#pragma unroll
      for (int k = 0; k < EACH / WIDE; ++k) {
        const uint4 raw = src[k * THREADS];
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (WIDE == 4) {
            x[4 * k + j] = __uint_as_float(w[j]);
          } else {
            x[8 * k + 2 * j] = __uint_as_float(w[j] << 16);
            x[8 * k + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
          }
        }
      }
      if (there < PIECE) {  // (whole pieces of 16 bytes are there)
#pragma unroll
        for (int k = 0; k < EACH; ++k)
          if (WIDE * (tid + k / WIDE * THREADS) >= there) x[k] = -INFINITY;
      }
    } else {
      const T* src = (const T*)a.logits + (size_t)row * a.stride + first;
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const int at = WIDE * (tid + k / WIDE * THREADS) + k % WIDE;
        x[k] = at < there ? to_f32(src[at]) : -INFINITY;
      }
    }
    // (fmaxf leaves NaN out)
    float tops4[EACH / 4], mine = -INFINITY;
#pragma unroll
    for (int k = 0; k < EACH / 4; ++k) {
      tops4[k] = fmaxf(max3(x[4 * k], x[4 * k + 1], x[4 * k + 2]), x[4 * k + 3]);
      mine = fmaxf(mine, tops4[k]);
    }
    const float top = unordered(__reduce_max_sync(0xffffffffu, ordered(mine)));  // of the warp
    // exponentials: the difference is exact or nearly so, and the error of a product with log2 e shrinks with the term
    float2 sums2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < EACH; k += 2) {
      const float2 y = mul2(add2(make_float2(x[k], x[k + 1]), make_float2(-top, -top)), make_float2(1.4426950408889634f, 1.4426950408889634f));
      sums2[k / 2 % 2] = add2(sums2[k / 2 % 2], make_float2(ex2_of(y.x), ex2_of(y.y)));
    }
    sums2[0] = add2(sums2[0], sums2[1]);
    float sum = sums2[0].x + sums2[0].y;
    if (!(sum < INFINITY)) {  // there is a NaN, or an infinity less itself: NaN counts as -inf, and infinities share the mass
      sum = 0.f;
#pragma unroll
      for (int k = 0; k < EACH; ++k)
        if (x[k] == x[k] && x[k] > -INFINITY) sum += x[k] == top ? 1.f : ex2_of((x[k] - top) * 1.4426950408889634f);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) a.stats[(size_t)p * WARPS + warp] = make_float2(top, sum);
    if (fresh) {
      // (each warp whose lanes all have logits vouches for an equal part of the wanted; where there are too few of them, none does)
      const int whole = max(1, min(WARPS, there / (32 * WIDE))), each = whole == WARPS ? (n + WARPS - 1) / WARPS : (n + whole - 1) / whole;
      const uint32_t kth = each <= 32 ? warp_kth(ordered(mine), each - 1) : NOTHING;
      if (lane == 0) bounds[warp] = warp < whole ? kth : 0xffffffffu;
      for (int i = tid; i < n; i += THREADS) list[i] = 0;
      if (tid == 0) found = n;
      aside = n;
      __syncthreads();
      limit = 0xffffffffu;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) limit = min(limit, bounds[w]);
      // what reaches the bound exceeds the number below it (that is not -0, which is none below 0); -inf does not
      limit = max(limit, NOTHING + 1) - 1;
      if (limit == 0x7fffffffu) --limit;
    }
    // what exceeds the limit (NaN does not); of equals the first column counts, and that was there before
    const float above = unordered(limit);
    if (mine > above) {
#pragma unroll
      for (int k = 0; k < EACH / 4; ++k) {
        if (!(tops4[k] > above)) continue;
#pragma unroll
        for (int j = 4 * k; j < 4 * k + 4; ++j) {
          if (x[j] > above) {
            const int at = atomicAdd(&found, 1);
            const uint32_t column = first + WIDE * (tid + j / WIDE * THREADS) + j % WIDE;
            if (at < LIST_CAP) list[at] = (unsigned long long)ordered(x[j]) << 32 | ~column;
          }
        }
      }
    }
    if (__syncthreads_or(!ok)) {  // a copy did not arrive: the block leaves together
      if (tid == 0) atomicOr(a.err, DSP_ERR_WAIT_LIMIT);
      // the parts that are left have no entries (the groups' kernel goes by what stands there)
      const int last_row = (end - 1) / a.pieces;
      for (int r = row + tid; r <= last_row; r += THREADS) a.parts[blockIdx.x + r] = (uint32_t)r << 16;
      if (tid == 0 && end % a.pieces == 0) a.parts[blockIdx.x + last_row + 1] = (uint32_t)last_row << 16;
      // let copies that are still on their way land before the shared memory goes away
#pragma unroll 1
      for (int i = 0; i < 2000; ++i) __nanosleep(100);
      return;
    }
    if (tid == 0) ask(p + STAGES, turn % STAGES);  // (everybody has this stage in registers)
    const bool last = ++in_row == a.pieces || p + 1 == end;
    int count = found;
    __syncthreads();  // (nobody puts anything aside before all have read that)
    if (count > LIST_CAP) {
      float copy[EACH];  // (so that the usual way keeps its registers)
#pragma unroll
      for (int k = 0; k < EACH; ++k) copy[k] = x[k];
      exact_bound<WIDE>(copy, limit, n, first, list, aside, &found, of_warp);
      count = found;
      __syncthreads();
    }
    aside = count;
    if (fresh || last || count > n + ASIDE) {
      unsigned long long* next = list == lists[0] ? lists[1] : lists[0];
      for (int i = tid; i < n; i += THREADS) next[i] = 0;
      __syncthreads();
      for (int i = tid; i < count; i += THREADS) {
        const unsigned long long key = list[i];
        if (key == 0) continue;
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += list[j] > key;  // (no two are equal: columns differ)
        if (rank < n) next[rank] = key;
      }
      if (tid == 0) found = n;
      aside = n;
      list = next;
      __syncthreads();
      limit = max((uint32_t)(list[n - 1] >> 32), NOTHING);
    }
    fresh = false;
    if (last) {
      int entries = 0;
      const int part = blockIdx.x + row;
      for (int i = tid; i < n; i += THREADS) {
        a.lists[(size_t)part * n + i] = list[i];
        entries += list[i] != 0;
      }
      entries = block_sum(entries, of_warp);
      if (tid == 0) {
        a.parts[part] = (uint32_t)row << 16 | (uint32_t)entries;
        if (in_row == a.pieces && p + 1 == end) a.parts[part + 1] = (uint32_t)row << 16;
      }
      if (in_row == a.pieces) {
        in_row = 0;
        ++row;
      }
      fresh = true;
    }
  }
}

// A candidate of a group: its key in order, its row (counted from the group's first) and column.
struct Candidate {
  unsigned long long key;
  uint32_t row, column;
  __device__ __forceinline__ bool before(const Candidate& o) const {
    return key > o.key || (key == o.key && (row < o.row || (row == o.row && column < o.column)));
  }
};

__global__ void __launch_bounds__(THREADS)
beam_groups_kernel(const Args a) {
  __shared__ Candidate list[CAP];
  __shared__ uint2 range[WARPS];
  __shared__ int reached[2][WARPS];
  __shared__ int open[CAP];  // lists whose first entry reaches the bound
  __shared__ int found, opened;
  __shared__ Candidate best_of_warp[WARPS], taken;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n, group = blockIdx.x;
  if (a.rows == 0) pdl_wait();  // (else the kernel in front was behind its own wait when this one began)
  const int first = a.group_start[group], end = a.group_start[group + 1];
  int* parent = a.parent + (size_t)group * n;
  int* token = a.token + (size_t)group * n;
  float* score = a.score + (size_t)group * n;
  const bool sound = first >= 0 && end >= first && end <= a.rows;
  if (!sound && tid == 0) atomicOr(a.err, DSP_ERR_BAD_GROUP);
  const int rows = sound ? end - first : 0;
  for (int i = tid; i < n; i += THREADS) {
    parent[i] = token[i] = -1;
    score[i] = -INFINITY;
  }
  if (tid == 0) found = opened = 0;
  pdl_launch_dependents();
  pdl_wait();
  // the rows' largest logits and sums: a warp a row
  const int per_row = a.pieces * WARPS;
  for (int r = warp; r < rows; r += WARPS) {
    const float2* stats = a.stats + (size_t)(first + r) * per_row;
    float top = -INFINITY;
    for (int i = lane; i < per_row; i += 32) top = fmaxf(top, stats[i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.;
    for (int i = lane; i < per_row; i += 32) {
      const float2 of = stats[i];
      if (of.x == top)
        sum += (double)of.y;
      else if (of.x > -INFINITY && top < INFINITY)
        sum += (double)of.y * exp((double)of.x - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) a.of_rows[first + r] = make_float2(top, (float)log(sum));
  }
  __syncthreads();
  auto first_cta = [&](int r) { return r * a.pieces / a.run; };
  auto last_cta = [&](int r) { return (r * a.pieces + a.pieces - 1) / a.run; };
  // the parts of the group's rows follow one another
  const int part0 = rows > 0 ? first_cta(first) + first : 0, lists = rows > 0 ? last_cta(end - 1) + end - part0 : 0;
  auto entries = [&](int l) -> int {
    const uint32_t row_count = a.parts[part0 + l];
    return isfinite(a.scores[row_count >> 16]) ? (int)(row_count & 0xffffu) : 0;
  };
  auto candidate = [&](int l, int depth) -> Candidate {
    const int row = (int)(a.parts[part0 + l] >> 16);
    const unsigned long long e = a.lists[(size_t)(part0 + l) * n + depth];
    const float x = unordered((uint32_t)(e >> 32));
    const float2 of_row = a.of_rows[row];
    const double away = x == of_row.x ? 0. : (double)x - (double)of_row.x;
    return {ordered((double)a.scores[row] + away - (double)of_row.y), (uint32_t)(row - first), ~(uint32_t)e};
  };
  // A lower bound of the n-th best key, in its first 32 bits.  Of each list (they are in order) every `each`-th entry is looked at,
  // some 1,024 in all, four a thread; an entry that is at least t stands for `each` that are, so that ceil(n / each) of them
  // vouch for n.  The largest such t is bisected to a 4,096th of what lies between the best and the worst.
  const int each = min(n, (lists * n + SAMPLES - 1) / SAMPLES), per_list = each > 0 ? n / each : 0;
  uint32_t sample[SAMPLES / THREADS];
#pragma unroll
  for (int k = 0; k < SAMPLES / THREADS; ++k) {
    sample[k] = (uint32_t)(NOTHING64 >> 32);
    if (lists <= SAMPLES) {
      const int i = tid + k * THREADS, l = i / max(per_list, 1), depth = (i - l * per_list + 1) * each - 1;
      if (l < lists && depth < entries(l)) sample[k] = (uint32_t)(candidate(l, depth).key >> 32);
    } else {  // the best of several lists' first entries
      for (int l = tid + k * THREADS; l < lists; l += SAMPLES)
        if (entries(l) > 0) sample[k] = max(sample[k], (uint32_t)(candidate(l, 0).key >> 32));
    }
  }
  const int wanted = lists <= SAMPLES ? (n + max(each, 1) - 1) / max(each, 1) : n;
  constexpr uint32_t NONE = (uint32_t)(NOTHING64 >> 32);
  uint32_t lo = 0xffffffffu, hi = NONE;
  int there = 0;
#pragma unroll
  for (int k = 0; k < SAMPLES / THREADS; ++k) {
    if (sample[k] > NONE) {
      ++there;
      lo = min(lo, sample[k]);
    }
    hi = max(hi, sample[k]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  there = __reduce_add_sync(0xffffffffu, there);
  if (lane == 0) {
    range[warp] = make_uint2(lo, hi);
    reached[1][warp] = there;
  }
  __syncthreads();
  there = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    lo = min(lo, range[w].x);
    hi = max(hi, range[w].y);
    there += reached[1][w];
  }
  if (there < wanted) lo = hi = NONE;  // everything is let through
#pragma unroll 1
  for (int step = 0; step < 12 && lo < hi; ++step) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    int c = 0;
#pragma unroll
    for (int k = 0; k < SAMPLES / THREADS; ++k) c += sample[k] >= mid;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) reached[step & 1][warp] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) c += reached[step & 1][w];
    if (c >= wanted)
      lo = mid;
    else
      hi = mid - 1;
  }
  const uint32_t limit = lo;
  auto reaches = [&](const Candidate& c) { return (uint32_t)(c.key >> 32) >= limit && c.key > NOTHING64; };
  for (int l = tid; l < lists; l += THREADS)
    if (entries(l) > 0 && reaches(candidate(l, 0))) {
      const int at = atomicAdd(&opened, 1);
      if (at < CAP) open[at] = l;
    }
  __syncthreads();
  // the entries of those lists, side by side
  for (int i = tid; i < min(opened, CAP) * n; i += THREADS) {
    const int l = open[i / n], depth = i % n;
    if (depth >= entries(l)) continue;
    const Candidate c = candidate(l, depth);
    if (!reaches(c)) continue;
    const int at = atomicAdd(&found, 1);
    if (at < CAP) list[at] = c;
  }
  __syncthreads();
  if (found <= CAP && opened <= CAP) {
    const int count = found;
    for (int i = tid; i < count; i += THREADS) {
      const Candidate c = list[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += list[j].before(c);
      if (rank < n) {
        parent[rank] = first + (int)c.row;
        token[rank] = (int)c.column;
        score[rank] = (float)unordered(c.key);
      }
    }
    return;
  }
  // too many reach it (many equal keys): the best one is taken, then the best behind it, and so on
  for (int i = 0; i < n; ++i) {
    Candidate best = {NOTHING64, 0xffffffffu, 0xffffffffu};
    for (int l = tid; l < lists; l += THREADS) {
      // the first of the list that comes behind the one taken last (a list is in order)
      int lo = 0, hi = entries(l);
      while (i > 0 && lo < hi) {
        const int mid = (lo + hi) / 2;
        if (taken.before(candidate(l, mid)))
          hi = mid;
        else
          lo = mid + 1;
      }
      if (lo < entries(l)) {
        const Candidate c = candidate(l, lo);
        if (c.key > NOTHING64 && c.before(best)) best = c;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Candidate other = {__shfl_xor_sync(0xffffffffu, best.key, o), __shfl_xor_sync(0xffffffffu, best.row, o),
                               __shfl_xor_sync(0xffffffffu, best.column, o)};
      if (other.before(best)) best = other;
    }
    if (lane == 0) best_of_warp[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < WARPS; ++w)
        if (best_of_warp[w].before(best)) best = best_of_warp[w];
      taken = best;
      if (best.key > NOTHING64) {
        parent[i] = first + (int)best.row;
        token[i] = (int)best.column;
        score[i] = (float)unordered(best.key);
      }
    }
    __syncthreads();
  }
}

// Floats of scratch, and where its arrays begin.
long layout(Args& a, float* at, long rows, long pieces, long ctas, long n) {
  a.lists = reinterpret_cast<unsigned long long*>(at);
  a.stats = reinterpret_cast<float2*>(a.lists + (rows + ctas) * n);
  a.of_rows = a.stats + rows * pieces * WARPS;
  a.parts = reinterpret_cast<uint32_t*>(a.of_rows + rows);
  return (rows + ctas) * (2 * n + 1) + 2 * rows * (pieces * WARPS + 1);
}
}  // namespace

// tensors: logits, scores, group_start, parent, token, score, scratch
extern "C" int dsp_beam_select(const DspTensor* t, cudaStream_t stream) {
  const DspTensor &logits = t[0], &scores = t[1], &start = t[2], &parent = t[3], &token = t[4], &score = t[5], &scratch = t[6];
#define SELECT_REQUIRE(cond, ...) DSP_REQUIRE(cond, "beam_select: " __VA_ARGS__)
  SELECT_REQUIRE(logits.device >= 0, "CUDA tensors only (there is no CPU path)");
  SELECT_REQUIRE(logits.dims == 2 && (logits.dtype == DSP_T_F32 || logits.dtype == DSP_T_BF16), "logits [R, V] in float32 or bfloat16 expected");
  const long R = logits.size[0], V = logits.size[1];
  SELECT_REQUIRE(V <= 1 || logits.stride[1] == 1, "neighbouring logits of a row must lie side by side");
  SELECT_REQUIRE(start.dims == 1 && start.size[0] >= 1, "group_start must be one-dimensional and have an end");
  const long groups = start.size[0] - 1, n = parent.dims == 2 ? parent.size[1] : 0;
  SELECT_REQUIRE(n >= 1 && n <= MAX_COUNT, "count %ld must be 1 to %d", n, MAX_COUNT);
  SELECT_REQUIRE(V >= 1 && V <= 0x7fffffff - PIECE && R <= 65535 && groups <= 0x7fffffff, "%ld rows of %ld logits: at most 65535 rows", R, V);
  SELECT_REQUIRE(tensor_is(scores, DSP_T_F32, logits.device, 1, R), "scores must be contiguous float32 [%ld] on the device of the logits", R);
  SELECT_REQUIRE(tensor_is(start, DSP_T_I32, logits.device, 1, groups + 1), "group_start must be contiguous int32 on the device of the logits");
  SELECT_REQUIRE(tensor_is(parent, DSP_T_I32, logits.device, 2, groups, n) && tensor_is(token, DSP_T_I32, logits.device, 2, groups, n) &&
                     tensor_is(score, DSP_T_F32, logits.device, 2, groups, n),
                 "results [%ld, %ld] expected", groups, n);
  if (groups == 0) return 0;
  SELECT_REQUIRE((uintptr_t)logits.data % (logits.dtype == DSP_T_F32 ? 4 : 2) == 0, "logits must be aligned to their size");
  SELECT_REQUIRE(current_device() == logits.device, "the tensors are on device %d, the current device is %d", logits.device, current_device());
  const int sms = dsp_num_sms();
  const long pieces = (V + PIECE - 1) / PIECE, most_ctas = (sms > 0 ? sms : 1) * PIECES_CTAS;
  const long run = max((R * pieces + most_ctas - 1) / most_ctas, 1L), ctas = (R * pieces + run - 1) / run;
  SELECT_REQUIRE(R * pieces <= 1 << 30, "%ld rows of %ld logits are too many for one call", R, V);
  Args a = {};
  const long need = layout(a, (float*)scratch.data, R, pieces, ctas, n);
  SELECT_REQUIRE(scratch.contiguous && scratch.device == logits.device && scratch.dims == 1 && scratch.dtype == DSP_T_F32 &&
                     (uintptr_t)scratch.data % 16 == 0 && scratch.size[0] >= need,
                 "scratch is too small");
  a.logits = logits.data;
  a.scores = (const float*)scores.data;
  a.group_start = (const int*)start.data;
  a.parent = (int*)parent.data;
  a.token = (int*)token.data;
  a.score = (float*)score.data;
  a.stride = R > 1 ? logits.stride[0] : 0;
  a.rows = (int)R;
  a.groups = (int)groups;
  a.vocab = (int)V;
  a.pieces = (int)pieces;
  a.run = (int)run;
  a.n = (int)n;
  a.err = dsp_device_error_ptr();
  SELECT_REQUIRE(a.err != nullptr, "no device error word");
  if (R > 0) {
    const bool f32 = logits.dtype == DSP_T_F32;
    const long size = f32 ? 4 : 2;
    a.bulk = (uintptr_t)logits.data % 16 == 0 && a.stride * size % 16 == 0 && V * size % 16 == 0;
    const size_t smem = a.bulk ? STAGES * PIECE * size : 0;
    const dim3 grid((unsigned)ctas);
    auto go = [&](auto kernel) -> int {
      static bool allowed[2][MAX_DEVICES] = {};  // asked for once a device and type
      const int device = current_device();
      if (device < 0 || !allowed[f32][device]) {
        DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(STAGES * PIECE * size)));
        if (device >= 0) allowed[f32][device] = true;
      }
      DSP_CUDA(launch_pdl(kernel, grid, dim3(THREADS), smem, stream, a));
      return 0;
    };
    const int rc = f32 ? go(beam_pieces_kernel<float>) : go(beam_pieces_kernel<bf16>);
    if (rc != 0) return rc;
  }
  DSP_CUDA(launch_pdl(beam_groups_kernel, dim3((unsigned)groups), dim3(THREADS), 0, stream, a));
  DSP_CHECK_LAUNCH("beam_select");
  return 0;
}
