// The best continuations of every group of beams.
//
// Row r has logits x_v and a score s_r so far; group g has the rows group_start[g] .. group_start[g + 1] - 1.  Its candidates are
// (r, v) with
//     key(r, v) = s_r + (x_v - max x) - log sum_v exp(x_v - max x)
// in 64 bits, the logarithm rounded to 32 (so that equal rows have equal keys, whatever the order of a sum).  Wanted are the n
// largest keys in descending order, ties to the lowest row, then the lowest v.  NaN counts as -inf; what is -inf is no
// candidate; a row whose score is not finite has none; where infinities are the largest logits, they share the mass.
//
// Within a row the order of keys is that of logits, so the n best of a piece of a row can be told before its sum is known.
// One pass over the logits: a block holds 8,192 of a row in registers, 32 a thread, and leaves their maximum, their sum of
// exponentials and their n best in order.  A lower bound of the n-th best, which few others reach, costs no
// search: of each of the 8 warps the ceil(n / 8)-th largest of its lanes' maxima, of these the smallest: at least n logits are as
// large.  What reaches it (some 2 n) is put in order by counting.  Where too many do (many equal logits), the exact bound is
// bisected.  A block a group then merges the sums of its rows' pieces and picks n of the pieces' lists in the same way.
//
// Loads bound it.
#include "packed2.cuh"
#include "tensor_checks.cuh"

namespace {
constexpr int THREADS = 256, WARPS = THREADS / 32, EACH = 32, PIECE = THREADS * EACH;
constexpr int MAX_COUNT = 8 * 32;  // each warp vouches for an eighth of the wanted
constexpr int CAP = 1024;          // candidates that are put in order by counting

// Statistics of a piece of a row and how many entries its list has.
struct Stat {
  double sum;  // of exp(x - top)
  float top;
  int count;
};

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
template <typename K>
__device__ __forceinline__ K warp_kth(K x, int k) {
  const int lane = threadIdx.x & 31;
  if constexpr (sizeof(K) == 4) {
    if (k < 4) {  // one after the other is quicker
      for (int i = 0; i < k; ++i) {
        const uint32_t those = __ballot_sync(0xffffffffu, x == __reduce_max_sync(0xffffffffu, x));
        if (lane == __ffs(those) - 1) x = 0;
      }
      return __reduce_max_sync(0xffffffffu, x);
    }
  }
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const K y = __shfl_xor_sync(0xffffffffu, x, step);
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
  Stat* stats;                  // [rows][pieces]
  unsigned long long* lists;    // [rows][pieces][n]: logit in order and its column's complement
  float2* of_rows;              // [rows] largest logit and logarithm of the sum
  long stride;                  // of a row of logits
  int rows, groups, vocab, pieces, n;
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

// Where more logits reach the lower bound than can be put in order: the n-th largest by bisection, and where its equals are more
// than wanted, the last column taken.  By the whole block; how many are in the list then.
template <int WIDE>
__device__ __noinline__ int exact_bound(const float* x, uint32_t bound, uint32_t all_top, int n, int first, unsigned long long* list,
                                        int* found, int* of_warp) {
  const int tid = threadIdx.x;
  uint32_t lo = bound, hi = all_top;  // at least n are >= lo (or all that there are); the answer is in lo .. hi
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
  if (tid == 0) *found = 0;
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < EACH; ++k) {
    const int column = WIDE * (tid + k / WIDE * THREADS) + k % WIDE;
    const uint32_t o = ordered(x[k]);
    if ((o > lo || (o == lo && column <= c0)) && x[k] > -INFINITY) {
      const int at = atomicAdd(found, 1);
      if (at < CAP) list[at] = (unsigned long long)o << 32 | ~(uint32_t)(first + column);
    }
  }
  __syncthreads();
  return min(*found, CAP);
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 4)
beam_pieces_kernel(const Args a) {
  __shared__ unsigned long long list[CAP];
  __shared__ double sums[WARPS];
  __shared__ uint32_t tops[WARPS], bounds[WARPS];
  __shared__ int of_warp[WARPS], found;
  constexpr int WIDE = 16 / sizeof(T);  // logits of a load
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
  const int row = blockIdx.y, first = blockIdx.x * PIECE;
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: the next kernel looks at the groups before it waits)
  if (tid == 0) found = 0;
  // Thread t has the columns first + WIDE (t + 256 k) .. + WIDE - 1, however the row lies in memory: equal rows give equal sums.
  const T* src = (const T*)a.logits + (size_t)row * a.stride + first;
  float x[EACH];
  const int there = a.vocab - first;  // columns from this block's first on
  if (there >= PIECE && (uintptr_t)src % 16 == 0) {
    uint4 raw[EACH / WIDE];
#pragma unroll
    for (int k = 0; k < EACH / WIDE; ++k) raw[k] = __ldcs(reinterpret_cast<const uint4*>(src) + tid + k * THREADS);
#pragma unroll
    for (int k = 0; k < EACH / WIDE; ++k) {
      const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
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
  } else {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int at = WIDE * (tid + k / WIDE * THREADS) + k % WIDE;
      x[k] = at < there ? to_f32(src[at]) : -INFINITY;
    }
  }
  // (fmaxf leaves NaN out)
  float tops4[EACH / 4], top = -INFINITY;
#pragma unroll
  for (int k = 0; k < EACH / 4; ++k) {
    tops4[k] = fmaxf(max3(x[4 * k], x[4 * k + 1], x[4 * k + 2]), x[4 * k + 3]);
    top = fmaxf(top, tops4[k]);
  }
  const float mine = top;
  const uint32_t kth = warp_kth(ordered(top), (n + WARPS - 1) / WARPS - 1);
  const uint32_t warp_top = __reduce_max_sync(0xffffffffu, ordered(top));
  if (lane == 0) {
    tops[warp] = warp_top;
    bounds[warp] = kth;
  }
  __syncthreads();
  uint32_t all_top = 0, bound = 0xffffffffu;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    all_top = max(all_top, tops[w]);
    bound = min(bound, bounds[w]);
  }
  top = unordered(all_top);
  // what reaches the bound (NaN does not)
  const float limit = unordered(max(bound, NOTHING));
  if (mine >= limit && mine > -INFINITY) {
#pragma unroll
    for (int k = 0; k < EACH / 4; ++k) {
      if (!(tops4[k] >= limit)) continue;
#pragma unroll
      for (int j = 4 * k; j < 4 * k + 4; ++j) {
        if (x[j] >= limit && x[j] > -INFINITY) {
          const int at = atomicAdd(&found, 1);
          const uint32_t column = first + WIDE * (tid + j / WIDE * THREADS) + j % WIDE;
          if (at < CAP) list[at] = (unsigned long long)ordered(x[j]) << 32 | ~column;
        }
      }
    }
  }
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
  double all = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  if (lane == 0) sums[warp] = all;
  __syncthreads();
  int count = found;
  if (count > CAP) {
    float copy[EACH];  // (so that the usual way keeps its registers)
#pragma unroll
    for (int k = 0; k < EACH; ++k) copy[k] = x[k];
    count = exact_bound<WIDE>(copy, bound, all_top, n, first, list, &found, of_warp);
  }
  const size_t piece = (size_t)row * a.pieces + blockIdx.x;
  unsigned long long* out = a.lists + piece * n;
  for (int i = tid; i < count; i += THREADS) {
    const unsigned long long key = list[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += list[j] > key;  // (no two are equal: columns differ)
    if (rank < n) out[rank] = key;
  }
  if (tid == 0) {
    double total = 0.;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += sums[w];
    a.stats[piece] = {total, top, min(count, n)};
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
  __shared__ uint4 heads[THREADS / 4];
  __shared__ int open[CAP];  // lists whose first entry reaches the bound
  __shared__ uint32_t bound;
  __shared__ int found, opened;
  __shared__ Candidate best_of_warp[WARPS], taken;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n, group = blockIdx.x;
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
  if (tid == 0) {
    found = opened = 0;
    bound = (uint32_t)(NOTHING64 >> 32);
  }
  pdl_launch_dependents();
  pdl_wait();
  // the rows' largest logits and sums: a warp a row
  for (int r = warp; r < rows; r += WARPS) {
    const Stat* stats = a.stats + (size_t)(first + r) * a.pieces;
    float top = -INFINITY;
    for (int p = lane; p < a.pieces; p += 32) top = fmaxf(top, stats[p].top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.;
    for (int p = lane; p < a.pieces; p += 32) {
      const float of = stats[p].top;
      if (of == top)
        sum += stats[p].sum;
      else if (of > -INFINITY && top < INFINITY)
        sum += stats[p].sum * exp((double)of - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) a.of_rows[first + r] = make_float2(top, (float)log(sum));
  }
  __syncthreads();
  const int lists = rows * a.pieces;
  auto entries = [&](int l) -> int {
    const int r = first + l / a.pieces;
    const float s = a.scores[r];
    return isfinite(s) ? a.stats[(size_t)first * a.pieces + l].count : 0;
  };
  auto candidate = [&](int l, int depth) -> Candidate {
    const int r = l / a.pieces;
    const unsigned long long e = a.lists[((size_t)first * a.pieces + l) * n + depth];
    const float x = unordered((uint32_t)(e >> 32));
    const float2 of_row = a.of_rows[first + r];
    const double away = x == of_row.x ? 0. : (double)x - (double)of_row.x;
    return {ordered((double)a.scores[first + r] + away - (double)of_row.y), (uint32_t)r, ~(uint32_t)e};
  };
  // A lower bound of the n-th best key, in its first 32 bits: the n-th of 256, a candidate a thread or the best of a thread's lists.
  unsigned long long mine = NOTHING64;
  if (lists >= THREADS) {
    for (int l = tid; l < lists; l += THREADS)
      if (entries(l) > 0) mine = max(mine, candidate(l, 0).key);
  } else if (lists > 0) {
    const int l = tid % lists, depth = tid / lists;
    if (depth < entries(l)) mine = candidate(l, depth).key;
  }
  const uint32_t head = (uint32_t)(mine >> 32);
  reinterpret_cast<uint32_t*>(heads)[tid] = head;
  __syncthreads();
  int larger = 0;
  for (int j = 0; j < THREADS / 4; ++j) {
    const uint4 x = heads[j];
    // (equals in the order of the threads: one of them is the n-th)
    larger += (x.x > head || (x.x == head && 4 * j < tid)) + (x.y > head || (x.y == head && 4 * j + 1 < tid)) +
              (x.z > head || (x.z == head && 4 * j + 2 < tid)) + (x.w > head || (x.w == head && 4 * j + 3 < tid));
  }
  if (larger == n - 1) bound = head;
  __syncthreads();
  const uint32_t limit = bound;
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

long scratch_bytes(long rows, long pieces, long n) {
  return rows * pieces * (long)(sizeof(Stat) + 8 * n) + rows * (long)sizeof(float2);
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
  const long pieces = (V + PIECE - 1) / PIECE;
  SELECT_REQUIRE(R * pieces <= 0x7fffffff, "%ld rows of %ld logits are too many for one call", R, V);
  SELECT_REQUIRE(scratch.contiguous && scratch.device == logits.device && scratch.dims == 1 && scratch.dtype == DSP_T_F32 &&
                     (uintptr_t)scratch.data % 16 == 0 && scratch.size[0] * 4 >= scratch_bytes(R, pieces, n),
                 "scratch is too small");
  Args a = {};
  a.logits = logits.data;
  a.scores = (const float*)scores.data;
  a.group_start = (const int*)start.data;
  a.parent = (int*)parent.data;
  a.token = (int*)token.data;
  a.score = (float*)score.data;
  a.stats = reinterpret_cast<Stat*>(scratch.data);
  a.lists = reinterpret_cast<unsigned long long*>(a.stats + R * pieces);
  a.of_rows = reinterpret_cast<float2*>(a.lists + R * pieces * n);
  a.stride = R > 1 ? logits.stride[0] : 0;
  a.rows = (int)R;
  a.groups = (int)groups;
  a.vocab = (int)V;
  a.pieces = (int)pieces;
  a.n = (int)n;
  a.err = dsp_device_error_ptr();
  SELECT_REQUIRE(a.err != nullptr, "no device error word");
  if (R > 0) {
    const dim3 grid((unsigned)pieces, (unsigned)R);
    if (logits.dtype == DSP_T_F32)
      DSP_CUDA(launch_pdl(beam_pieces_kernel<float>, grid, dim3(THREADS), 0, stream, a));
    else
      DSP_CUDA(launch_pdl(beam_pieces_kernel<bf16>, grid, dim3(THREADS), 0, stream, a));
  }
  DSP_CUDA(launch_pdl(beam_groups_kernel, dim3((unsigned)groups), dim3(THREADS), 0, stream, a));
  DSP_CHECK_LAUNCH("beam_select");
  return 0;
}
