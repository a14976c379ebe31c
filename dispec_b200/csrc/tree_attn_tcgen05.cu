// Attention of drafted trees over the paged cache on the fifth-generation tensor cores, bfloat16 in, 32-bit softmax and
// accumulation (the formula: tree_attn.cu; how the work is cut: tree_schedule.cuh).  Compiled once per head size
// (-DDSP_HEAD_DIM=64 or 128).
//
// One CTA an SM walks its run of units: for each item's share, 128 query rows of one key/value head and key tiles of 64.
// S = Q K^T and O += P V are tcgen05.mma with S, O and the A operands Q and P in tensor memory; keys and values arrive by
// TMA in rings of their own that run on from share to share.  Roles:
//   warp 0      requests the key and value tiles;
//   warps 1, 11 issue the score products of softmax group 0 and of group 1;
//   warp 10     issues the output products;
//   warps 2..9  two softmax groups of four warps: group g owns the key tiles g, g + 2, ... of a share with a score buffer,
//               output accumulator, P, running maximum and sum of its own; thread r of a group owns row r.
// The whole block meets once a share.  Behind that barrier the softmax warps put the share's queries down, which they asked for
// before it, then merge the two halves of the last one and store its rows (or leave a partial result); warp 0 has worked the
// share out and asked for its first tiles before.  What a row sees of a tile that holds nodes of the tree is a mask of 64 bits, cut from
// its words of `visible`.  Value rows that no row of the item may see are zeroed in shared memory before the output product, and
// so are, in tiles that not every row sees whole, values that are not finite, which a weight of 0 would carry to rows that do
// not see them: behind the product they are added to the rows that do.  Every wait is bounded; one that runs out sets the
// device error word.
//
// What bounds it: not bytes and not the tensor pipe (512 of 1,200 cycles a key tile), but the softmax groups' chain per tile: scores
// out of tensor memory, maximum, 64 exponentials a thread, weights back.  64 trees of 64 nodes behind 2,050 tokens, 40 heads of 128
// on 8: 232 us, 0.55 PFLOP/s with the rows there are and 2.2 TB/s; 2 trees of 24 behind 32,768, 28 on 4: 52 us, 2.3 TB/s.  Two groups
// of one row a thread: the accumulators, scores, weights and queries of 128 rows then fill tensor memory, and a third group, or
// key tiles of 128, has no room beside them (queries in shared memory and weights in the place of their scores would make
// some; that was not tried).
#include "tcgen05_common.cuh"
#include "tree_schedule.cuh"

#ifndef DSP_HEAD_DIM
#error "compile with -DDSP_HEAD_DIM=<head size>"
#endif
#define DSP_CAT2(a, b) a##b
#define DSP_CAT(a, b) DSP_CAT2(a, b)

namespace {
using namespace tc;
using namespace tree;

constexpr int D = DSP_HEAD_DIM;
static_assert(D == 64 || D == 128, "this kernel is built for head sizes 64 and 128");
constexpr int BM = 1 << ROW_SHIFT_TENSOR_CORES, BN = KEYS_PER_TILE, THREADS = 384;
// Key tiles of a share go to two issuing warps in turn, and each waits for its own tiles only.  With an even ring the tiles of a
// share in one slot all belong to one of them; with an odd one a warp that is ahead (its tile landed, an older one of the
// other's has not) could take the slot's last phase but one for the phase it waits for.  From share to share a slot may change
// hands (behind an odd number of tiles): the block meets in between, when every tile of the last share has landed and been
// used, and that barrier is needed for it.
constexpr int K_STAGES = 6, V_STAGES = 6;
static_assert(K_STAGES % 2 == 0, "in a share, a slot of the key ring belongs to one issuing warp");
constexpr int SHARES = 4;      // the shares remembered: the next two, the present one and the one whose rows are being stored
constexpr int BAD_SLOTS = 16;  // a tile's unreadable pages are remembered until its softmax has begun
static_assert(BAD_SLOTS >= K_STAGES + 4, "a slot is rewritten K_STAGES + 4 tiles later at the earliest");
constexpr int PV_WARP = 10, S1_WARP = 11;
constexpr int KD = D / 64;
// A tile in shared memory lies as the pages are brought (tcgen05_common.cuh): [group of 8 keys][slice of 64 columns][8 rows of 128
// bytes], a page's rows in one TMA request.
constexpr int SLICE = KEY_SLICE;
constexpr int GROUP = KD * SLICE;
constexpr int KV_BYTES = BN / 8 * GROUP;
constexpr int SMEM_BYTES = (K_STAGES + V_STAGES) * KV_BYTES + 1024;
// tensor memory, 32-bit columns
constexpr int S_COLS = BN;
constexpr int O_COL = 2 * S_COLS;
constexpr int P_COLS = BN / 2;
constexpr int P_COL = O_COL + 2 * D;
constexpr int Q_COL = P_COL + 2 * P_COLS;
constexpr int TMEM_COLS = 512;
static_assert(Q_COL + D / 2 <= TMEM_COLS, "tensor memory layout");
// Of eight weights, so many are formed on the multiply-add pipe: 64 trees of 64 nodes behind 2,050 tokens, 40 heads of 128 on 8:
// 240 us with none, 232 with two, 237 with three; 2 trees of 24 behind 32,768 on scattered pages 50.7 with none and 52.0 with two,
// 8 trees of 16 the same with both.  The larger call decides.  The result's error is the same to four digits (2.305e-3 of its size
// against 64 bits, 2.342e-3 behind 32,768).  Heads of 64, with half of the products to a weight: no difference, none.
constexpr int EX2_FMA = D == 128 ? 2 : 0;
constexpr float RESCALE_STEP = 8.f;  // the running maximum follows the true one in steps of 2^8

// Two bfloat16 values: one that is not finite; the same with 0 in its place.
__device__ __forceinline__ bool has_odd(uint32_t x) { return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t without_odd(uint32_t x) {
  return ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u);
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

struct Params {
  DspTreeAttention a;
  int page_runs;  // the run maps are valid
  float scale_log2;
};

// Which keys key0 .. key0 + 63 the row of a node sees: stored ones, and nodes of the tree by the row's words.
__device__ __forceinline__ unsigned long long seen_keys(const Params& p, const Share& t, int row, int depth, int key0) {
  unsigned long long stored = 0ull, drafted = 0ull;
  const int off = key0 - t.ctx;  // number of the first key as a node
  if (off < 0) {
    stored = off <= -64 ? ~0ull : (1ull << -off) - 1ull;
    if (p.a.sh.window > 0) {
      const int hidden = t.ctx + depth - p.a.sh.window + 1 - key0;  // so many first keys are out of the window
      if (hidden > 0) stored = hidden >= 64 ? 0ull : stored & ~((1ull << hidden) - 1ull);
    }
  }
  if (off > -64 && off < t.n) {
    const unsigned long long* w = p.a.visible + (size_t)row * p.a.words;
    if (off <= 0) {
      drafted = w[0] << -off;
    } else {
      const int k = off >> 6, sft = off & 63;
      drafted = k < p.a.words ? w[k] >> sft : 0ull;
      if (sft && k + 1 < p.a.words) drafted |= w[k + 1] << (64 - sft);
    }
    const int there = t.n - off;  // keys up to the tree's last node
    if (there < 64) drafted &= (1ull << there) - 1ull;
    if (p.a.sh.window > 0 && depth >= p.a.sh.window) {  // a tree deeper than the window
#pragma unroll 1
      for (unsigned long long left = drafted; left != 0ull; left &= left - 1ull) {
        const int c = __ffsll((long long)left) - 1;
        if (p.a.depth[t.first + off + c] <= depth - p.a.sh.window) drafted &= ~(1ull << c);
      }
    }
  }
  return stored | drafted;
}

// By the 128 threads of a group, two a key: value rows that no row of the item may see become zeros (whole 128-byte rows, every
// slice), and so do, in tiles that not every row sees whole, numbers that are not finite.  True: there was such a number in this
// thread's half of a key that some row may see.
__device__ __forceinline__ bool clean_values(const Params& p, const Share& t, uint32_t tile_addr, int tile, uint32_t bad, int r) {
  const int key_row = r >> 1, key = tile * BN + key_row, window = p.a.sh.window;
  const bool dead = key >= t.ctx + t.n || (window > 0 && key <= t.ctx - window) ||
                    ((bad >> (key_row >> (__ffs(p.a.page_size) - 1))) & 1u);
  const uint32_t row_addr = tile_addr + (uint32_t)(key_row >> 3) * GROUP + (uint32_t)(key_row & 7) * 128u + (uint32_t)(r & 1) * 64u;
  const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
  bool any = false;
#pragma unroll 1
  for (int h = 0; h < KD; ++h) {
    const uint32_t at = row_addr + h * SLICE;
    uint4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = dead ? make_uint4(0, 0, 0, 0) : ld_shared16(at + c * 16);
    // 0 times a number that is not finite is NaN, and so is every sum with it
    __nv_bfloat162 sum = zero;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]), zero, sum);
    }
    const bool found = has_odd(*reinterpret_cast<const uint32_t*>(&sum));
    if (!found && !dead) continue;
    any |= found;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      st_shared16(at + c * 16, make_uint4(without_odd(v[c].x), without_odd(v[c].y), without_odd(v[c].z), without_odd(v[c].w)));
  }
  fence_async_smem();
  return any;
}

// By a whole warp, behind its group's last output product of a share: the values that clean_values took out of the group's tiles
// are added to the rows that see their keys, in their own columns (a weight is positive, and changes nothing in what is not
// finite).  They are read again where they lie, which costs nothing until there are some.  (A function of its own: its code
// stays out of the way.)
__device__ __noinline__ void add_odd_values(const Params& p, const Share& t, int g, int node, bool row_ok, uint32_t o_addr) {
  const Shape& sh = p.a.sh;
  const int* table = p.a.page_table + (size_t)t.seq * p.a.pt_stride;
  const int depth = sh.window > 0 ? p.a.depth[node] : 0;
#pragma unroll 1
  for (int tile = t.kt_begin + g; tile < t.kt_end; tile += 2) {
    const int key0 = tile * BN;
    auto page_of = [&](int key) {
      const int place = key / p.a.page_size, page = place < p.a.table_width ? table[place] : -1;
      return page < p.a.num_pages ? page : -1;
    };
    // as in the walk: tiles that not every row sees whole, or with a page that is not there
    bool cleaned = key0 > t.ctx - BN || (sh.window > 0 && key0 <= t.ctx + t.n - 1 - sh.window);
#pragma unroll 1
    for (int c = 0; c < BN; c += p.a.page_size) cleaned |= page_of(key0 + c) < 0;
    if (!cleaned) continue;
    const unsigned long long seen = row_ok ? seen_keys(p, t, node, depth, key0) : 0ull;
#pragma unroll 1
    for (int c = 0; c < BN; ++c) {
      const bool mine = (seen >> c) & 1ull;
      const int page = page_of(key0 + c);
      if (page < 0 || !__any_sync(0xffffffffu, mine)) continue;
      const bf16* v = (const bf16*)p.a.v_pool + (((size_t)page * sh.KVH + t.head) * p.a.page_size + (key0 + c) % p.a.page_size) * D;
      bool found = false;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) found |= !isfinite(__bfloat162float(v[c0 + (threadIdx.x & 31)]));
      if (!__any_sync(0xffffffffu, found)) continue;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t ov[32];
        tmem_ld32(o_addr + (uint32_t)c0, ov);
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float x = __bfloat162float(v[c0 + k]);
          if (mine && !isfinite(x)) ov[k] = __float_as_uint(__uint_as_float(ov[k]) + x);
        }
        __syncwarp();
        tmem_st32(o_addr + (uint32_t)c0, ov);
        tmem_st_wait();
      }
    }
  }
}

// a * b + c and a + b of two numbers at once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x of two numbers up to 2^7 or so on the multiply-add pipe: x = n + f, n whole, |f| <= 1/2; 2^f by a polynomial of degree 3
// (interpolation at the Chebyshev points of the interval: below 1.1e-4 off, a twentieth of the bfloat16 rounding of a
// weight), times 2^n from n's bits, which are 0 at x <= -127.  -inf gives 0, NaN stays.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  constexpr float C0 = 0.99992454f, C1 = 0.69313675f, C2 = 0.24263948f, C3 = 0.05583828f;
  constexpr float WHOLE = 12583039.f;  // 1.5 * 2^23 + 127: the sum's last bits are n + 127
  x = make_float2(max_nan(x.x, -127.f), max_nan(x.y, -127.f));
  const float2 t = add2(x, make_float2(WHOLE, WHOLE));
  const float2 n = add2(t, make_float2(-WHOLE, -WHOLE));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 y = fma2(f, make_float2(C3, C3), make_float2(C2, C2));
  y = fma2(y, f, make_float2(C1, C1));
  y = fma2(y, f, make_float2(C0, C0));
  return mul2(y, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}

// Four lanes' pieces change hands: piece k of the j-th of four neighbouring lanes becomes piece j of the k-th.
__device__ __forceinline__ void transpose4(uint4 (&x)[4]) {
#pragma unroll
  for (int s = 1; s < 4; s <<= 1) {
    const bool up = threadIdx.x & s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & s) continue;
      uint4 v = up ? x[i] : x[i | s];
      v.x = __shfl_xor_sync(0xffffffffu, v.x, s);
      v.y = __shfl_xor_sync(0xffffffffu, v.y, s);
      v.z = __shfl_xor_sync(0xffffffffu, v.z, s);
      v.w = __shfl_xor_sync(0xffffffffu, v.w, s);
      if (up)
        x[i] = v;
      else
        x[i | s] = v;
    }
  }
}

// Multiplies a row's accumulators by alpha.
__device__ __forceinline__ void rescale(uint32_t o_addr, float alpha) {
#pragma unroll 1
  for (int c0 = 0; c0 < D; c0 += 32) {
    uint32_t ov[32];
    tmem_ld32(o_addr + (uint32_t)c0, ov);
#pragma unroll
    for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
    tmem_st32(o_addr + (uint32_t)c0, ov);
  }
}

__global__ void __launch_bounds__(THREADS, 1)
tree_attn_tcgen05_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap runs_k,
                         const __grid_constant__ CUtensorMap runs_v) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);  // swizzle atoms are 1024 bytes
  __shared__ __align__(8) uint64_t k_full[K_STAGES], k_empty[K_STAGES];  // landed; its scores are complete
  __shared__ __align__(8) uint64_t v_full[V_STAGES], v_empty[V_STAGES];  // landed; its output product is complete
  __shared__ __align__(8) uint64_t s_full[2], s_free[2];  // a score buffer is complete; the group has read it
  __shared__ __align__(8) uint64_t p_full[2], o_done[2];  // P written, O rescaled, V rows zeroed; the output product is complete
  __shared__ __align__(8) uint64_t q_ready[2];            // the queries of a share with tiles for the group are in tensor memory
  __shared__ __align__(8) uint64_t o_free;                // the last share's accumulators have been read
  __shared__ float2 merge_ml[2][2][BM];                   // a group's maximum and sum per row, by share in turn
  __shared__ Share shares[SHARES];                        // share k in k % SHARES, written by warp 0 in share k - 2 or before
  __shared__ int odd_share[2];  // the last share in which a group took numbers out of the values
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;        // a wait ran out
  __shared__ int failed_share;  // the first share in which one did: the block leaves together behind that share's barrier
  __shared__ uint32_t bad_pages[BAD_SLOTS];  // of key tile n, in slot n % BAD_SLOTS; bit j: page j had no valid id (not loaded)

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Shape& sh = p.a.sh;
  const int G = sh.G;
  unsigned char* k_s = smem;  // [stage] tiles
  unsigned char* v_s = k_s + K_STAGES * KV_BYTES;

  pdl_wait();
  Walk w;  // warp 0's, a share ahead
  bool more = false;
  auto step = [&](int share) {  // works that share out, the one behind the last
    const Split split = w.split(sh);
    more = w.next(sh);
    if (lane == 0) {
      if (!more) {
        w.at.seq = -1;
        p.a.scratch.splits[w.cta] = split;
      }
      shares[share % SHARES] = w.at;
    }
    __syncwarp();
  };
  if (warp == 0) {
    more = w.begin(sh, blockIdx.x, gridDim.x);
    if (lane == 0) {
      if (!more) {
        w.at.seq = -1;
        p.a.scratch.splits[w.cta].parts = 0;
      }
      shares[0] = w.at;
    }
    if (more) step(1);
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tid == 64) {
    for (int s = 0; s < K_STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < V_STAGES; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&s_free[b], 4);
      mbar_init(&p_full[b], 4);
      mbar_init(&o_done[b], 1);
    }
    mbar_init(&q_ready[0], D == 128 ? 8 : 4);
    mbar_init(&q_ready[1], D == 128 ? 8 : 4);
    mbar_init(&o_free, 8);
    failed = 0;
    failed_share = 0x7fffffff;
    odd_share[0] = odd_share[1] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  auto give_up = [&](int share) {
    failed = 1;
    atomicMin(&failed_share, share);
  };

  int done = 0;   // key tiles of the shares before
  int share = 0;
  // warp 0: ring slots of the next tile, and their use counts; tiles of the coming share that have been asked for
  int sk = 0, rk = 0, sv = 0, rv = 0, asked = 0;
  int pg = -2, pg_next = -2;                                // the page ids of a chunk of tiles, and of the next one
  uint32_t bad_mask = 0, live_mask = 0, run_mask = 0;
  // warps 1, 10, 11: shares of the group with tiles, tiles of each group
  int active = 0, count0 = 0, count1 = 0;
  // softmax warps: the group's tiles so far, running maximum and sum of the present share
  int count = 0;
  float m_run = -INFINITY, l_run = 0.f;
  const bool leader = elect_one();

  // Rows of tile `quarter` of the softmax warps.
  const int g = warp >= 2 && warp < PV_WARP ? (warp - 2) >> 2 : warp == S1_WARP ? 1 : 0;  // the group of warps 1 to 9 and 11
  const int quarter = warp & 3, r = quarter * 32 + lane;
  const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);

  // Requests the tiles asked .. upto - 1 of a share, two a turn (`upto` is even or the share's last).
  auto request = [&](const Share& t, int upto, int first_tile) {
    const int pages_per_tile = BN / p.a.page_size, groups = p.a.page_size >> 3;
    const uint32_t page_bytes = (uint32_t)KD * (uint32_t)p.a.page_size * 128u;
    const int ppt_shift = __ffs(pages_per_tile) - 1, page_shift = __ffs(p.a.page_size) - 1;  // powers of two here
    const int chunk_shift = 5 - ppt_shift, chunk_mask = (1 << chunk_shift) - 1;
    const int page_in_tile = lane & (pages_per_tile - 1);
    const uint32_t tile_lanes = pages_per_tile == 32 ? 0xffffffffu : ((1u << pages_per_tile) - 1u);
    const int n_kt = t.kt_end - t.kt_begin, kt_begin = t.kt_begin, head = t.head;
    const int lo = sh.window > 0 ? max(0, t.ctx - sh.window + 1) : 0, last = t.ctx + t.n - 1;
    const int* table = p.a.page_table + (size_t)t.seq * p.a.pt_stride;
    // Page ids are looked up for a chunk of 32 / pages_per_tile tiles at a time, a chunk ahead.
    auto load_chunk = [&](int c) -> int {
      const int i = (c << chunk_shift) + (lane >> ppt_shift);
      const int first = (kt_begin + i) * BN + page_in_tile * p.a.page_size;
      if (i < n_kt && first <= last && first + p.a.page_size > lo) {
        const int j = first >> page_shift;
        return j < p.a.table_width ? table[j] : -1;
      }
      return -2;  // not wanted
    };
    if (asked == 0) pg_next = load_chunk(0);
#pragma unroll 1
    for (; asked < upto; asked += 2) {
      const int in_chunk = asked & chunk_mask;
      if (in_chunk == 0) {
        pg = pg_next;
        pg_next = load_chunk((asked >> chunk_shift) + 1);
        const bool bad = pg != -2 && (pg < 0 || pg >= p.a.num_pages);  // recorded, not loaded, its keys are hidden
        if (bad) {
          atomicOr(p.a.err, DSP_ERR_BAD_PAGE);
          pg = -1;
        }
        bad_mask = __ballot_sync(0xffffffffu, bad);
        live_mask = __ballot_sync(0xffffffffu, pg >= 0);
        const int first_pg = __shfl_sync(0xffffffffu, pg, lane & ~(pages_per_tile - 1));
        run_mask = __ballot_sync(0xffffffffu, pg >= 0 && pg == first_pg + page_in_tile &&
                                                  first_pg + pages_per_tile <= p.a.num_pages);
      }
      // Two tiles per turn, each with a lane of its own that waits for the tile's ring slots and makes the requests.
      const int second = (lane >> ppt_shift) - in_chunk;  // 0, 1: this lane holds a page of the turn's first, second tile
      const bool mine = (second == 0 || second == 1) && asked + second < n_kt;
      const int shift = (in_chunk + (second == 1 ? 1 : 0)) << ppt_shift;
      const uint32_t live = (live_mask >> shift) & tile_lanes;
      const bool in_run = p.page_runs && ((run_mask >> shift) & tile_lanes) == tile_lanes;
      int my_sk = sk, my_rk = rk, my_sv = sv, my_rv = rv;
      if (second == 1) {
        if (++my_sk == K_STAGES) {
          my_sk = 0;
          ++my_rk;
        }
        if (++my_sv == V_STAGES) {
          my_sv = 0;
          ++my_rv;
        }
      }
      if (mine && lane == shift) {
        if (*(volatile int*)&failed == 0 &&
            mbar_wait_both(&k_empty[my_sk], (my_rk & 1) ^ 1, &v_empty[my_sv], (my_rv & 1) ^ 1)) {
          bad_pages[(first_tile + asked + second) % BAD_SLOTS] = (bad_mask >> shift) & tile_lanes;  // published by the arrival on k_full
          if (live == 0) {
            mbar_arrive(&k_full[my_sk]);
            mbar_arrive(&v_full[my_sv]);
          } else {
            mbar_expect_tx(&k_full[my_sk], (uint32_t)__popc(live) * page_bytes);
            mbar_expect_tx(&v_full[my_sv], (uint32_t)__popc(live) * page_bytes);
          }
          if (in_run) {  // the tile's pages lie one after the other in the pool: one request per operand
            load_pages(k_s + my_sk * KV_BYTES, &runs_k, &k_full[my_sk], head * groups, pg);
            load_pages(v_s + my_sv * KV_BYTES, &runs_v, &v_full[my_sv], head * groups, pg);
          }
        } else {
          give_up(share);
        }
      }
      if (!__all_sync(0xffffffffu, !mine || in_run)) {
        if (mine && !in_run && pg >= 0 && *(volatile int*)&failed == 0) {
          const int dst = page_in_tile * groups * GROUP;
          load_pages(k_s + my_sk * KV_BYTES + dst, &map_k, &k_full[my_sk], head * groups, pg);
          load_pages(v_s + my_sv * KV_BYTES + dst, &map_v, &v_full[my_sv], head * groups, pg);
        }
      }
#pragma unroll 1
      for (int u = 0; u < min(2, n_kt - asked); ++u) {
        if (++sk == K_STAGES) {
          sk = 0;
          ++rk;
        }
        if (++sv == V_STAGES) {
          sv = 0;
          ++rv;
        }
      }
    }
  };

  // Rows in global memory: a lane holds a row of the tile, but four neighbouring lanes read and write 64 bytes of each of their
  // rows together (a row a lane, 16 bytes each, an instruction touches 32 lines: 3.5 us from a share's end to the next one's
  // queries).  Where the four lanes' rows begin in a tensor of rows (node, head); `n` of them are there.
  const int r4 = r & ~3;
  struct Rows4 {
    size_t at[4];
    int n;
  };
  auto rows_of = [&](const Share& t, size_t stride) -> Rows4 {
    Rows4 x;
    const int first = t.row_tile * BM + r4;
    int node = first / G, head = first - node * G;
    x.n = min(4, t.n * G - first);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x.at[k] = (size_t)(t.first + node) * stride + (size_t)(t.head * G + head) * D;
      if (++head == G) {
        head = 0;
        ++node;
      }
    }
    return x;
  };

  // The queries of a share: row r of the tile, lane r, two bfloat16 per column (rows past the item are zero).  In heads of 128
  // each group brings half of the columns, in heads of 64 group 1 brings them all.  Asked for first, put down later.
  constexpr int Q_PIECES = 8;  // of 16 bytes, a lane
  auto ask_queries = [&](const Share& t, bool wanted, uint4 (&x)[Q_PIECES]) {
    const Rows4 rows = rows_of(t, p.a.q_stride);
    const bf16* q = (const bf16*)p.a.q + (D == 128 ? g * 64 : 0) + (lane & 3) * 8;
#pragma unroll
    for (int c = 0; c < Q_PIECES; ++c)
      x[c] = wanted && c % 4 < rows.n ? __ldg(reinterpret_cast<const uint4*>(q + rows.at[c % 4] + c / 4 * 32)) : make_uint4(0, 0, 0, 0);
  };
  auto put_queries = [&](const Share& t, const uint4 (&x)[Q_PIECES]) {
    uint32_t y[32];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 z[4] = {x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]};
      transpose4(z);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        y[16 * h + 4 * c] = z[c].x;
        y[16 * h + 4 * c + 1] = z[c].y;
        y[16 * h + 4 * c + 2] = z[c].z;
        y[16 * h + 4 * c + 3] = z[c].w;
      }
    }
    __syncwarp();
    tmem_st32(lane_addr + (uint32_t)(Q_COL + (D == 128 ? g * 32 : 0)), y);
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&q_ready[0]);
      if (t.kt_end - t.kt_begin > 1) mbar_arrive(&q_ready[1]);
    }
  };

  // Behind the barrier of share k: merges the two groups' halves and stores the rows, or the partial result of the share; each
  // group has half of the columns.
  auto finish = [&](int k) {
    const Share& t = shares[k % SHARES];
    const int row0 = t.row_tile * BM, nrows = min(BM, t.n * G - row0), slot = t.slot;
    const bool row_ok = r < nrows;
    const bool two = t.kt_end - t.kt_begin > 1;
    const float2 ml0 = merge_ml[k & 1][0][r], ml1 = two ? merge_ml[k & 1][1][r] : make_float2(-INFINITY, 0.f);
    const float M = fmaxf(ml0.x, ml1.x);
    const float w0 = ml0.x == -INFINITY ? 0.f : ex2(ml0.x - M);
    const float w1 = ml1.x == -INFINITY ? 0.f : ex2(ml1.x - M);
    const float denom = ml0.y * w0 + ml1.y * w1;
    const float inv = slot >= 0 ? 1.f : denom == 0.f ? 0.f : 1.f / denom;
    const float f0 = w0 * inv, f1 = w1 * inv;
    if (quarter * 32 < nrows) {
      Rows4 rows;
      if (slot < 0) rows = rows_of(t, p.a.out_stride);
      bf16* out = (bf16*)p.a.out + (lane & 3) * 8;
      float* part = p.a.scratch.part_o + ((size_t)slot * BM + r4) * D + (lane & 3) * 4;
#pragma unroll 1
      for (int c0 = g * (D / 2); c0 < (g + 1) * (D / 2); c0 += 32) {
        uint32_t ov[32], ow[32];
        __syncwarp();
        tmem_ld32(lane_addr + (uint32_t)(O_COL + c0), ov);
        // (a half that saw no key has weight 0, and an accumulator of zeros)
        if (two) {
          tmem_ld32(lane_addr + (uint32_t)(O_COL + D + c0), ow);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            ov[c] = __float_as_uint(__uint_as_float(ov[c]) * f0 + __uint_as_float(ow[c]) * f1);
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * f0);
        }
        if (slot >= 0) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 x[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
              x[c] = make_uint4(ov[16 * h + 4 * c], ov[16 * h + 4 * c + 1], ov[16 * h + 4 * c + 2], ov[16 * h + 4 * c + 3]);
            transpose4(x);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (r4 + k < nrows) *reinterpret_cast<uint4*>(part + k * D + c0 + 16 * h) = x[k];
          }
        } else {
          uint4 x[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            x[c].x = pack2(__uint_as_float(ov[8 * c]), __uint_as_float(ov[8 * c + 1]));
            x[c].y = pack2(__uint_as_float(ov[8 * c + 2]), __uint_as_float(ov[8 * c + 3]));
            x[c].z = pack2(__uint_as_float(ov[8 * c + 4]), __uint_as_float(ov[8 * c + 5]));
            x[c].w = pack2(__uint_as_float(ov[8 * c + 6]), __uint_as_float(ov[8 * c + 7]));
          }
          transpose4(x);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < rows.n) *reinterpret_cast<uint4*>(out + rows.at[k] + c0) = x[k];
        }
        __syncwarp();
      }
      if (g == 0 && slot >= 0 && row_ok) reinterpret_cast<float2*>(p.a.scratch.part_ml)[(size_t)slot * BM + r] = make_float2(M, denom);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&o_free);
  };

  uint4 x[Q_PIECES];  // the coming queries
  const bool brings = D == 128 || g == 1;
  if (warp >= 2 && warp < PV_WARP) ask_queries(shares[0], brings && shares[0].seq >= 0, x);

  // Every wait of a share is for something that happens in that share, or, in warp 0's requests for the coming one, for
  // slots that this share's tiles leave; the whole block passes the barrier at its end.
#pragma unroll 1
  for (;; ++share) {
    const Share& t = shares[share % SHARES];
    const bool sound = failed_share >= share, another = sound && t.seq >= 0;  // (written before the last barrier; all see the same)
    if (!another) pdl_launch_dependents();
    if (warp >= 2 && warp < PV_WARP) {
      // the queries of this share, asked for before, and the end of the last one while its scores form
      if (another && brings) put_queries(t, x);
      if (share > 0 && sound) finish(share - 1);
    }
    if (!another) break;
    const int n_kt = t.kt_end - t.kt_begin;
    if (warp == 0) {
      // this share's tiles, then the coming one's first: as many as slots that this share's tiles are sure to leave
#pragma unroll 1
      for (int ahead = 0; ahead < 2; ++ahead) {
        const Share& of = shares[(share + ahead) % SHARES];
        if (of.seq < 0) break;
        const int tiles = of.kt_end - of.kt_begin;
        request(of, ahead ? min(K_STAGES - 2, tiles) : tiles, ahead ? done + n_kt : done);
        if (ahead) break;
        if (more) step(share + 2);
        asked = 0;
      }
    } else if (warp == 1 || warp == S1_WARP) {
      // ---- score products of one softmax group
      const uint32_t idesc_s = umma_idesc(BM, BN);
      const uint64_t k_desc0 = key_desc(smem_u32(k_s), GROUP);
      const uint32_t tmem_s = tmem_base + (uint32_t)(g * S_COLS);
      bool ok = true;
      if (g < n_kt) {
        ok = __all_sync(0xffffffffu, mbar_wait(&q_ready[g], active & 1));
        ++active;
        tc_fence_after();
      }
#pragma unroll 1
      for (int a = g; a < n_kt && ok; a += 2, ++count0) {
        const int s = (done + a) % K_STAGES, use = (done + a) / K_STAGES;
        ok = __all_sync(0xffffffffu, count0 == 0 ? mbar_wait(&k_full[s], use & 1)
                                                 : mbar_wait_both(&k_full[s], use & 1, &s_free[g], (count0 - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const uint64_t k_desc = k_desc0 + (uint64_t)(s * (KV_BYTES >> 4));
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (uint32_t)(k >> 2), in = (uint32_t)(k & 3) * 32u;
            umma_a_tmem(tmem_s, tmem_base + (uint32_t)(Q_COL + k * 8), k_desc + ((off * SLICE + in) >> 4), idesc_s, k != 0);
          }
          umma_commit(&s_full[g]);
          umma_commit(&k_empty[s]);
        }
        __syncwarp();
      }
      if (!ok) give_up(share);
    } else if (warp == PV_WARP) {
      // ---- output products: O[g] += P[g] V of the share's tiles in turn
      const uint32_t idesc_o = umma_idesc(BM, D) | (1u << 16);  // B (values) is N-major
      const uint64_t v_desc0 = value_desc(smem_u32(v_s), GROUP);
      bool ok = share == 0 || __all_sync(0xffffffffu, mbar_wait(&o_free, (share - 1) & 1));
#pragma unroll 1
      for (int b = 0; b < n_kt && ok; ++b) {
        const int og = b & 1, st = (done + b) % V_STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait_both(&v_full[st], ((done + b) / V_STAGES) & 1, &p_full[og],
                                                    (og ? count1 : count0) & 1));
        if (!ok) break;
        if (og)
          ++count1;
        else
          ++count0;
        tc_fence_after();
        const uint64_t v_desc = v_desc0 + (uint64_t)(st * (KV_BYTES >> 4));
        if (leader) {
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            umma_a_tmem(tmem_base + (uint32_t)(O_COL + og * D), tmem_base + (uint32_t)(P_COL + og * P_COLS + k * 8),
                        v_desc + (uint64_t)(k * (2 * GROUP >> 4)), idesc_o, (b >= 2) || k != 0);
          umma_commit(&v_empty[st]);
          umma_commit(&o_done[og]);
        }
        __syncwarp();
      }
      if (!ok) give_up(share);
    } else {
      // ---- softmax groups
      const uint32_t s_addr = lane_addr + (uint32_t)(g * S_COLS);
      const uint32_t o_addr = lane_addr + (uint32_t)(O_COL + g * D);
      const uint32_t p_addr = lane_addr + (uint32_t)(P_COL + g * P_COLS);
      const float scale = p.scale_log2;
      const int page_shift = __ffs(p.a.page_size) - 1;
      const int kt_begin = t.kt_begin, row0 = t.row_tile * BM;
      const int nrows = min(BM, t.n * G - row0);
      const bool row_ok = r < nrows;
      const bool warp_ok = quarter * 32 < nrows;  // a warp without rows only keeps the barriers going
      const int node = row_ok ? t.first + (row0 + r) / G : t.first;
      const int depth = sh.window > 0 ? p.a.depth[node] : 0;
      // tiles that begin between these are seen whole by every row (no node is deeper than the tree has nodes)
      const int all_before = t.ctx - BN, some_upto = sh.window > 0 ? t.ctx + t.n - 1 - sh.window : -1;
      const int lo_r = sh.window > 0 ? t.ctx + depth - sh.window + 1 : 0;
      m_run = -INFINITY;
      l_run = 0.f;
      bool ok = true;
      int j = 0;  // tiles of this group in this share
#pragma unroll 1
      for (int i = g; i < n_kt; i += 2, ++j, ++count) {
        const int key0 = (kt_begin + i) * BN;
        // what the row sees of a tile that not every row sees whole, while its scores are being formed
        const bool some = key0 > all_before || (sh.window > 0 && __any_sync(0xffffffffu, key0 < lo_r));
        unsigned long long seen = ~0ull;
        if (some && warp_ok) seen = row_ok ? seen_keys(p, t, node, depth, key0) : 0ull;
        // the tile's scores; and the group's previous O[g] += P V has to be complete before O[g] is rescaled and P[g] rewritten (no
        // arrival for a tile comes before every warp's for the one before has been counted)
        if (!__all_sync(0xffffffffu, j == 0 ? mbar_wait(&s_full[g], count & 1)
                                            : mbar_wait_both(&s_full[g], count & 1, &o_done[g], (count - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t bad = bad_pages[(done + i) % BAD_SLOTS];
        if (bad != 0u)
#pragma unroll 1
          for (int b = 0; b < BN >> page_shift; ++b)
            if ((bad >> b) & 1u)
              seen &= ~((p.a.page_size == 64 ? ~0ull : (1ull << p.a.page_size) - 1ull) << (b << page_shift));
        __syncwarp();
        if (warp_ok) {
          uint32_t a[32], b[32];
          tmem_ld32_nowait(s_addr, a);
          tmem_ld32_nowait(s_addr + 32, b);
          tmem_ld_wait();
          // the scores are in registers: the next scores of this group may overwrite S[g]
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[g]);
          if (some || bad != 0u) {
            const uint32_t s_lo = (uint32_t)seen, s_hi = (uint32_t)(seen >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              a[c] = (s_lo >> c) & 1u ? a[c] : 0xff800000u;  // -inf
              b[c] = (s_hi >> c) & 1u ? b[c] : 0xff800000u;
            }
          }
          float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            t0 = max3(t0, __uint_as_float(a[c]), __uint_as_float(a[c + 1]));
            t1 = max3(t1, __uint_as_float(a[c + 2]), __uint_as_float(a[c + 3]));
            t2 = max3(t2, __uint_as_float(b[c]), __uint_as_float(b[c + 1]));
            t3 = max3(t3, __uint_as_float(b[c + 2]), __uint_as_float(b[c + 3]));
          }
          const float tmax = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * scale;  // the scale is positive
          const float m_new = (tmax > m_run + RESCALE_STEP || m_run == -INFINITY) ? fmaxf(tmax, m_run) : m_run;
          const float alpha = m_new == m_run ? 1.f : ex2(m_run - m_new);  // 0 on a row's first visible tile
          m_run = m_new;
          const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
          // two scores an instruction where there is one for it
          const float2 scale2 = make_float2(scale, scale), neg_m2 = make_float2(neg_m, neg_m);
          float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(a[c]), __uint_as_float(a[c + 1])), scale2, neg_m2);
            const float2 y = fma2(make_float2(__uint_as_float(b[c]), __uint_as_float(b[c + 1])), scale2, neg_m2);
            const float2 ex = make_float2(ex2(x.x), ex2(x.y));
            const float2 ey = c / 2 % 4 < EX2_FMA ? ex2_fma(y) : make_float2(ex2(y.x), ex2(y.y));
            // the second product takes weights of eight bits, as it takes values (their sum is of the 32-bit ones): with both the
            // result is off by 2.3e-3 of its size, and by 1.65e-3 from its own rounding alone
            sum0 = add2(sum0, ex);
            sum1 = add2(sum1, ey);
            pk[c / 2] = pack2(ex.x, ex.y);
            pk[16 + c / 2] = pack2(ey.x, ey.y);
          }
          sum0 = add2(sum0, sum1);
          l_run = l_run * alpha + (sum0.x + sum0.y);
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) rescale(o_addr, alpha);
          __syncwarp();
          tmem_st32(p_addr, pk);  // 64 bfloat16 in the 32 columns of the group's A operand
        } else {
          if (lane == 0) mbar_arrive(&s_free[g]);
        }
        // values that 0 as a weight would not keep out
        if (key0 > all_before || key0 <= some_upto || bad != 0u) {
          const int st = (done + i) % V_STAGES;
          if (!__all_sync(0xffffffffu, mbar_wait(&v_full[st], ((done + i) / V_STAGES) & 1))) {
            ok = false;
            break;
          }
          if (clean_values(p, t, smem_u32(v_s + st * KV_BYTES), kt_begin + i, bad, r)) odd_share[g] = share;
        }
        __syncwarp();
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
      }
      const Share& next = shares[(share + 1) % SHARES];
      ask_queries(next, brings && next.seq >= 0, x);
      // the group's last product of the share
      if (ok && j > 0) {
        if (__all_sync(0xffffffffu, mbar_wait(&o_done[g], (count - 1) & 1))) {
          if (odd_share[g] == share && warp_ok) {  // (every warp of the group has arrived for that product)
            tc_fence_after();
            add_odd_values(p, t, g, node, row_ok, o_addr);
            __syncwarp();
            ask_queries(next, brings && next.seq >= 0, x);  // (asked for again: they need not live through the call)
          }
        } else {
          ok = false;
        }
      }
      if (!ok) give_up(share);
      merge_ml[share & 1][g][r] = make_float2(m_run, l_run);
    }
    done += n_kt;
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (failed) {
    if (threadIdx.x == 0) {
      atomicOr(p.a.err, DSP_ERR_WAIT_LIMIT);
      p.a.scratch.splits[w.cta].parts = 0;
    }
    // let copies that are still on their way land before the shared memory goes away
#pragma unroll 1
    for (int i = 0; i < 2000; ++i) __nanosleep(100);
  }
  tc_fence_after();
  __syncwarp();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

}  // namespace

// The arguments come checked from dsp_tree_attention (tree_attn.cu), which also launches the merge.  Returns 0, or: 1 launch
// failed, 4 the shared-memory opt-in or the tensor maps failed.
extern "C" int DSP_CAT(dsp_tree_attention_tcgen05_d, DSP_HEAD_DIM)(const DspTreeAttention* a, cudaStream_t stream) {
  const int page = a->page_size;
  Params p = {};
  p.a = *a;
  p.a.sh.min_units = 2;  // one tile for each softmax group
  p.scale_log2 = a->scale * 1.4426950408889634f;
  CUtensorMap map_k, map_v, runs_k, runs_v;
  if (!make_map_pages(&map_k, a->k_pool, a->num_pages, a->sh.KVH, page, D, 1) ||
      !make_map_pages(&map_v, a->v_pool, a->num_pages, a->sh.KVH, page, D, 1))
    return 4;
  // a pool of fewer pages than a key tile has gives no map of runs
  p.page_runs = make_map_pages(&runs_k, a->k_pool, a->num_pages, a->sh.KVH, page, D, BN / page) &&
                make_map_pages(&runs_v, a->v_pool, a->num_pages, a->sh.KVH, page, D, BN / page);
  if (!p.page_runs) {
    runs_k = map_k;
    runs_v = map_v;
  }
  static bool allowed[MAX_DEVICES] = {};  // asked for once a device
  const int device = current_device();
  if (device < 0 || !allowed[device]) {
    if (cudaFuncSetAttribute(tree_attn_tcgen05_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess)
      return 4;
    if (device >= 0) allowed[device] = true;
  }
  return launch_pdl(tree_attn_tcgen05_kernel, dim3((unsigned)a->ctas), dim3(THREADS), (size_t)SMEM_BYTES, stream, p, map_k, map_v,
                    runs_k, runs_v) == cudaSuccess
             ? 0
             : 1;
}
