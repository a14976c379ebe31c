// Attention of sequences with a shared beginning where few rows meet a key: each sequence's own keys (G rows), and shared
// beginnings of few sequences.  bfloat16 in, 32-bit softmax and accumulation (the formula: shared_attn.cu; how the work is cut:
// shared_schedule.cuh).  Compiled once per head size (-DDSP_HEAD_DIM=32, 64 or 128).
//
// Such a share is its keys' way from memory: 512 bytes a key and head of 128, for up to 64 rows.  So two CTAs an SM keep a ring
// of key tiles on its way that runs on from share to share (tiles of 64 keys, requested by TMA page by page, or in one request
// where pages follow one another), and while one is between two shares the other one reads.  A warp requests, four work:
// of 16, 32 or 64 rows (MT = 1, 2, 4 row tiles of 16) warp w has row tile w % MT and 16 MT of a tile's keys, with a running
// maximum, sum and accumulator of its own, so that no warp waits for another inside a share; at its end the 4 / MT warps
// of a row tile join theirs.  The products are mma.sync m16n8k16 (8 cycles each): 64 rows and keys take 1,024 cycles of an SM's
// tensor pipe where their tile takes 1,400 from memory, and sixteen rows would leave seven eighths of a tcgen05 tile of 128 empty,
// which puts its rows through tensor memory and the whole block through a barrier for every share.
//
// What bounds it: with sixteen rows the way from memory once it is full (148 sequences of 1,000 tokens, 28 heads of 128 on 4: 303 MB
// in 58 us behind 6 us in which the runs are found, 5.2 TB/s; 1,150 cycles a tile and CTA are work), with 33 to 64 rows its own
// instructions (3,100 cycles a tile and CTA for 35, 3,750 for 64: products 1,024, reads of keys and values by every row tile 1,024,
// the softmax between them): 8 groups of 5 behind 4,101 tokens, 28 heads on 4: 29.7 us, 60 MB.  In calls this short the beginnings
// count: 3.7 us until the runs are found, 3.5 until the first tile is there, 3 for the first steps' instructions.
// Heads of 32, 28 on 4: those 8 groups 25.4 us (103 in 32-bit arithmetic), 148 sequences of 1,000 tokens 35.2 (185); they have no kernel for
// many rows: 64 sequences of 40 heads on 8 behind 32,768 tokens 118 us (849).
// Tried and not kept: all 64 keys of a tile in one step (the same 3,750 cycles, and spills); fragments loaded a step ahead of their
// products (3,900); 200 registers a thread (three warps of an SM's quarter have 16,384 together: one CTA an SM, 43.6 us for those 8
// groups); the next share's queries asked for before a share's warps are joined, whose columns then overlap (31.4 us: while one CTA is
// between shares the other one works).
#pragma once
#include "shared_schedule.cuh"
#include "packed2.cuh"
#include "paged_tile.cuh"

namespace {
constexpr int FEW_SHIFT = ROW_SHIFT_FEW, FEW_ROWS = 1 << FEW_SHIFT, FEW_WARPS = 4, FEW_THREADS = 32 * (FEW_WARPS + 1);
constexpr int FEW_STAGES = D == 128 ? 3 : 6, FEW_CTAS_PER_SM = 2;
constexpr int JOIN_COLS = 16, JOIN_PITCH = JOIN_COLS + 4;  // columns joined at a time, and a row of them in shared memory
constexpr int JOIN_FLOATS = FEW_WARPS * 16 * JOIN_PITCH;    // of one of two buffers
constexpr int FEW_SMEM = FEW_STAGES * 2 * KV_BYTES + 2 * JOIN_FLOATS * 4 + 1024;
static_assert(sizeof(shared::Groups) <= FEW_STAGES * 2 * KV_BYTES, "the plan is made where the ring will be");
static_assert(FEW_CTAS_PER_SM * (FEW_SMEM + 4096) <= 228 * 1024, "shared memory");

struct FewParams {
  DspSharedAttention a;
  int page_runs;
  float scale_log2;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// By all working warps: they meet, and learn whether one of them says yes.
__device__ __forceinline__ bool any_warp(bool yes) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)yes), "n"(FEW_WARPS * 32)
      : "memory");
  return all != 0;
}
// Keys of a block of 16 from `at` on whose bits are set: 0xffff for a key, two keys a word.
__device__ __forceinline__ uint32_t key_mask(uint32_t alive, int at) {
  return ((alive >> at) & 1u ? 0xffffu : 0u) | ((alive >> (at + 1)) & 1u ? 0xffff0000u : 0u);
}

// A key tile in shared memory.
struct Tile {
  uint32_t k_s, v_s;
  int key0;
  uint32_t bad;  // bit j: page j is not there
  bool ragged;   // not every row sees all of it
};

// By a warp: its sixteen rows over NB blocks of sixteen keys of a tile, from block `block` on.
template <int NB>
__device__ __forceinline__ void few_step(const Tile& tl, const shared::Share& t, int block, int page_shift, float scale,
                                         const uint32_t (&q)[D / 16][4], const int (&lo)[2], const int (&hi)[2], float (&o)[D / 8][4],
                                         float (&m)[2], float (&l)[2]) {
  const int lane = threadIdx.x & 31, tq = lane & 3, m8 = lane >> 3, l8 = lane & 7;
  const int c0 = block * 16, key0 = tl.key0;
  if (key0 + c0 >= t.end || key0 + c0 + 16 * NB <= t.begin) return;
  float sc[2 * NB][4] = {};
  {
    // (two chains of products for each eight keys where there is one block only)
    float odd[NB == 1 ? 2 : 1][4] = {};
    constexpr int EACH = 4 / NB < D / 16 ? 4 / NB : D / 16;  // steps of 16 columns that are loaded together
#pragma unroll
    for (int k0 = 0; k0 < D / 16; k0 += EACH) {
      uint32_t b[NB][EACH][4];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int row = c0 + n * 16 + (m8 >> 1) * 8 + l8;
        const uint32_t base = tl.k_s + row_at(row);
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
          const int chunk = (k0 + k) * 2 + (m8 & 1);
          ldmatrix4(b[n][k], base + piece_at(chunk, l8));
        }
      }
#pragma unroll
      for (int k = 0; k < EACH; ++k)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          mma16(NB == 1 && (k & 1) ? odd[0] : sc[2 * n], q[k0 + k], b[n][k][0], b[n][k][1]);
          mma16(NB == 1 && (k & 1) ? odd[NB == 1 ? 1 : 0] : sc[2 * n + 1], q[k0 + k], b[n][k][2], b[n][k][3]);
        }
    }
    if (NB == 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sc[0][j] += odd[0][j];
        sc[1][j] += odd[NB == 1 ? 1 : 0][j];
      }
    }
  }
  uint32_t alive = 0xffffffffu;  // keys of the blocks that some row may see
  if (tl.ragged) {
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = c0 + c * 8 + tq * 2 + (j & 1), key = key0 + at, i = j >> 1;
        const bool seen = key >= lo[i] && key < hi[i] && !((tl.bad >> (at >> page_shift)) & 1u);
        sc[c][j] = seen ? sc[c][j] : -INFINITY;
      }
    const int at = c0 + lane;
    alive = __ballot_sync(0xffffffffu, lane < 16 * NB && key0 + at >= t.begin && key0 + at < t.end && !((tl.bad >> (at >> page_shift)) & 1u));
  }
  float alpha[2];
  uint32_t pk[NB][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float top = fmaxf(sc[0][2 * i], sc[0][2 * i + 1]);
#pragma unroll
    for (int c = 1; c < 2 * NB; ++c) top = max3(top, sc[c][2 * i], sc[c][2 * i + 1]);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * scale;  // the scale is positive
    const float m_new = top > m[i] + RESCALE_STEP || m[i] == -INFINITY ? fmaxf(top, m[i]) : m[i];
    alpha[i] = m_new == m[i] ? 1.f : ex2(m[i] - m_new);
    m[i] = m_new;
    const float neg = m_new == -INFINITY ? 0.f : -m_new;
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c) {
      const float e0 = ex2(fmaf(sc[c][2 * i], scale, neg)), e1 = ex2(fmaf(sc[c][2 * i + 1], scale, neg));
      sum += e0 + e1;
      // the second product takes weights of eight bits, as it takes values (their sum is of the 32-bit ones)
      pk[c >> 1][i + 2 * (c & 1)] = pack2(e0, e1);
    }
    l[i] = l[i] * alpha[i] + sum;
  }
  if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      o[n][0] *= alpha[0];
      o[n][1] *= alpha[0];
      o[n][2] *= alpha[1];
      o[n][3] *= alpha[1];
    }
  }
  // Values of keys that no row sees are left out.  So are, where some rows see a key and others do not, numbers that are not finite,
  // which a weight of 0 would carry to rows that do not see them; the rows that see them get them behind the product.
  const bool mixed = tl.ragged && (t.begin != t.all_begin || t.end != t.all_end);
  bool odd = false;
#pragma unroll
  for (int c = 0; c < NB; ++c) {
    const int row = c0 + c * 16 + (m8 & 1) * 8 + l8;
    const uint32_t base = tl.v_s + row_at(row);
    if (!tl.ragged) {
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        const int chunk = n * 2 + (m8 >> 1);
        uint32_t b[4];
        ldmatrix4_trans(b, base + piece_at(chunk, l8));
        mma16(o[2 * n], pk[c], b[0], b[1]);
        mma16(o[2 * n + 1], pk[c], b[2], b[3]);
      }
    } else {
      const uint32_t mask0 = key_mask(alive, c * 16 + tq * 2), mask1 = key_mask(alive, c * 16 + tq * 2 + 8);
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        const int chunk = n * 2 + (m8 >> 1);
        uint32_t b[4];
        ldmatrix4_trans(b, base + piece_at(chunk, l8));
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] &= j & 1 ? mask1 : mask0;
        if (mixed) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            odd |= has_odd(b[j]);
            b[j] = without_odd(b[j]);
          }
        }
        mma16(o[2 * n], pk[c], b[0], b[1]);
        mma16(o[2 * n + 1], pk[c], b[2], b[3]);
      }
    }
  }
  if (mixed && __any_sync(0xffffffffu, odd)) {
#pragma unroll 1
    for (int c = 0; c < 16 * NB; ++c) {
      if (!((alive >> c) & 1u)) continue;
      const int key = key0 + c0 + c, at = c0 + c;
      const bool sees0 = key >= lo[0] && key < hi[0], sees1 = key >= lo[1] && key < hi[1];
      const uint32_t line = tl.v_s + row_at(at) + (uint32_t)tq * 4u;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        uint32_t x;
        asm volatile("ld.shared.u32 %0, [%1];"
                     : "=r"(x)
                     : "r"(line + piece_at(n, at & 7))
                     : "memory");
        const float x0 = __uint_as_float(x << 16), x1 = __uint_as_float(x & 0xffff0000u);
        if (!isfinite(x0)) {
          o[n][0] += sees0 ? x0 : 0.f;
          o[n][2] += sees1 ? x0 : 0.f;
        }
        if (!isfinite(x1)) {
          o[n][1] += sees0 ? x1 : 0.f;
          o[n][3] += sees1 ? x1 : 0.f;
        }
      }
    }
  }
}

// Joins the 4 / MT warps of each of the share's MT row tiles, by all working warps, and puts the rows down: `out` and `out_ml` are
// those of row tid / 4 of the tile, or null.
template <int MT>
__device__ __forceinline__ void join_warps(float* join, float2 (&join_ml)[FEW_WARPS][16], const float (&o)[D / 8][4], const float (&m)[2],
                                           const float (&l)[2], float* out, float2* out_ml) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tq = lane & 3, r = tid >> 2;
  if (tq == 0) {
    join_ml[warp][gid] = make_float2(m[0], l[0]);
    join_ml[warp][gid + 8] = make_float2(m[1], l[1]);
  }
  any_warp(false);
  float f[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < FEW_WARPS; w += MT) top = fmaxf(top, join_ml[w + (warp & (MT - 1))][gid + 8 * i].x);
    f[i] = m[i] == -INFINITY ? 1.f : ex2(m[i] - top);  // (a warp that saw no key has sums of 0, or of NaN, which stay)
  }
  if (out_ml != nullptr && tq == 0) {
    float top = -INFINITY, all = 0.f;
#pragma unroll
    for (int w = 0; w < FEW_WARPS; w += MT) top = fmaxf(top, join_ml[w + (r >> 4)][r & 15].x);
#pragma unroll
    for (int w = 0; w < FEW_WARPS; w += MT) {
      const float2 ml = join_ml[w + (r >> 4)][r & 15];
      all += ml.x == -INFINITY ? ml.y : ml.y * ex2(ml.x - top);
    }
    *out_ml = make_float2(top, all);
  }
  // so many columns at a time, in two buffers in turn: every warp puts its part of them down, then a thread adds up four
  // neighbouring ones of a row
  const float* sums = join + ((r >> 4) * 16 + (r & 15)) * JOIN_PITCH + tq * 4;
  float* mine = join + (warp * 16 + gid) * JOIN_PITCH + tq * 2;
#pragma unroll
  for (int c = 0; c < D / JOIN_COLS; ++c) {
    const int buffer = (c & 1) * JOIN_FLOATS;
#pragma unroll
    for (int n = 0; n < JOIN_COLS / 8; ++n) {
      const float(&x)[4] = o[c * (JOIN_COLS / 8) + n];
      *reinterpret_cast<float2*>(mine + buffer + n * 8) = make_float2(x[0] * f[0], x[1] * f[0]);
      *reinterpret_cast<float2*>(mine + buffer + 8 * JOIN_PITCH + n * 8) = make_float2(x[2] * f[1], x[3] * f[1]);
    }
    any_warp(false);
    if (out != nullptr) {
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < FEW_WARPS; w += MT) {
        const float4 x = *reinterpret_cast<const float4*>(sums + buffer + w * 16 * JOIN_PITCH);
        sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
      }
      *reinterpret_cast<float4*>(out + c * JOIN_COLS + tq * 4) = sum;
    }
  }
}

__global__ void __launch_bounds__(FEW_THREADS, FEW_CTAS_PER_SM)
shared_attn_few_kernel(const __grid_constant__ FewParams p, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap runs_k,
                       const __grid_constant__ CUtensorMap runs_v) {
  typedef shared::Share Share;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* join = reinterpret_cast<float*>(ring + FEW_STAGES * 2 * KV_BYTES);  // [warp][16 rows][JOIN_PITCH]
  __shared__ __align__(8) uint64_t full[FEW_STAGES], empty[FEW_STAGES], known[8];
  __shared__ uint32_t bad_pages[FEW_STAGES];  // bit j: page j of the tile had no valid id (not loaded)
  // Share k in k % 8, told before its first tile is requested: every warp has left the tile a ring and one before that one, so
  // none is further behind than FEW_STAGES + 1 shares.
  __shared__ Share shares[8];
  __shared__ float2 join_ml[FEW_WARPS][16];
  __shared__ shared::Run run;
  static_assert(FEW_STAGES + 1 < 8, "shares that a warp may still read");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const shared::Shape& sh = p.a.sh;
  const int G = sh.G;
  if (tid == 0) {
    for (int s = 0; s < FEW_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], FEW_WARPS);
    }
    for (int k = 0; k < 8; ++k) mbar_init(&known[k], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Behind the kernel for many rows, which was behind its own wait when this one began, nothing that is read here is still being written,
  // and the results lie apart: the wait is for the end (the merge waits for this kernel alone).
  if (!p.a.beside) pdl_wait();
  shared::make_plan(sh, *reinterpret_cast<shared::Groups*>(ring), run, blockIdx.x, gridDim.x);
  fence_async_smem();  // (the ring's memory was written by threads, and TMA writes it next)
  __syncthreads();
  const int page_size = p.a.page_size, page_shift = __ffs(page_size) - 1;

  if (warp == FEW_WARPS) {
    // ---- requests
    shared::Walk w;
    bool more = w.begin(sh, run, blockIdx.x), ok = true;
    const int pages_per_tile = BN >> page_shift, ppt_shift = 6 - page_shift, chunk_tiles = 32 >> ppt_shift;
    const int page_in_tile = lane & (pages_per_tile - 1);
    const uint32_t tile_lanes = (1u << pages_per_tile) - 1u;  // (at most eight pages)
    const uint32_t page_bytes = (uint32_t)page_size * D * 2;
    // ids of the pages of 32 / pages_per_tile tiles from tile kt on, lane by lane (-2: not wanted)
    auto load_chunk = [&](const Share& t, int kt) -> int {
      const int tile = kt + (lane >> ppt_shift), first = tile * BN + page_in_tile * page_size;
      if (tile >= t.kt_end || first >= t.end || first + page_size <= t.begin) return -2;
      const int j = first >> page_shift;
      return j < p.a.table_width ? max(p.a.page_table[(size_t)t.seq * p.a.pt_stride + j], -1) : -1;
    };
    int share = 0, tile = 0, pg_first = more ? load_chunk(w.at, w.at.kt_begin) : -2;
    while (more && ok) {
      const Share t = w.at;
      if (lane == 0) {
        shares[share & 7] = t;
        mbar_arrive(&known[share & 7]);
      }
      const shared::Note note = w.split(sh);
      int pg_next = pg_first;
      more = w.next(sh);
      if (lane == 0) SharedWork::note(p.a, w.cta, note, more);
      if (more) pg_first = load_chunk(w.at, w.at.kt_begin);  // (they arrive while this share's tiles are requested)
      int pg = -2;
      uint32_t bad_mask = 0, live_mask = 0, run_mask = 0;
#pragma unroll 1
      for (int kt = t.kt_begin; kt < t.kt_end; ++kt, ++tile) {
        const int in_chunk = (kt - t.kt_begin) & (chunk_tiles - 1);
        if (in_chunk == 0) {
          pg = pg_next;
          pg_next = load_chunk(t, kt + chunk_tiles);
          const bool bad = pg != -2 && (pg < 0 || pg >= p.a.num_pages);  // recorded, not loaded, its keys are hidden
          if (bad) {
            atomicOr(p.a.err, DSP_ERR_BAD_PAGE);
            pg = -1;
          }
          bad_mask = __ballot_sync(0xffffffffu, bad);
          live_mask = __ballot_sync(0xffffffffu, pg >= 0);
          const int first_pg = __shfl_sync(0xffffffffu, pg, lane & ~(pages_per_tile - 1));
          run_mask = __ballot_sync(0xffffffffu, pg >= 0 && pg == first_pg + page_in_tile && first_pg + pages_per_tile <= p.a.num_pages);
        }
        const int shift = in_chunk << ppt_shift, s = tile % FEW_STAGES;
        const uint32_t live = (live_mask >> shift) & tile_lanes;
        const bool in_run = p.page_runs && ((run_mask >> shift) & tile_lanes) == tile_lanes;
        ok = tile < FEW_STAGES || mbar_wait(&empty[s], (tile / FEW_STAGES - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        unsigned char *k_s = ring + s * 2 * KV_BYTES, *v_s = k_s + KV_BYTES;
        if (lane == 0) {
          bad_pages[s] = (bad_mask >> shift) & tile_lanes;  // published by the arrival
          if (live == 0)
            mbar_arrive(&full[s]);
          else
            mbar_expect_tx(&full[s], 2u * (uint32_t)__popc(live) * page_bytes);
        }
        __syncwarp();
        if (lane >> ppt_shift == in_chunk) {
          const int groups = page_size >> 3, dst = page_in_tile * groups * GROUP;
          if (in_run) {
            if (page_in_tile == 0) {
              load_pages(k_s, &runs_k, &full[s], t.head * groups, pg);
              load_pages(v_s, &runs_v, &full[s], t.head * groups, pg);
            }
          } else if (pg >= 0) {
            load_pages(k_s + dst, &map_k, &full[s], t.head * groups, pg);
            load_pages(v_s + dst, &map_v, &full[s], t.head * groups, pg);
          }
        }
      }
      ++share;
    }
    if (lane == 0 && ok) {  // the end
      shares[share & 7].seq = -1;
      mbar_arrive(&known[share & 7]);
    }
    pdl_launch_dependents();
    if (p.a.beside) pdl_wait();
    if (!ok) {
      if (lane == 0) atomicOr(p.a.err, DSP_ERR_WAIT_LIMIT);
      // let copies that are still on their way land before the shared memory goes away
#pragma unroll 1
      for (int i = 0; i < 2000; ++i) __nanosleep(100);
    }
    return;
  }

  // ---- work
  const int gid = lane >> 2, tq = lane & 3;
  const float scale = p.scale_log2;
  int tile = 0;
#pragma unroll 1
  for (int share = 0;; ++share) {
    bool ok = __all_sync(0xffffffffu, mbar_wait(&known[share & 7], (share >> 3) & 1));
    const Share& t = shares[share & 7];
    const bool ended = !ok || t.seq < 0;
    const int row0 = t.row_tile << FEW_SHIFT, nrows = min(FEW_ROWS, t.n * G - row0), head = t.head;
    const int MT = nrows <= 16 ? 1 : nrows <= 32 ? 2 : 4;
    const int first_block = warp / MT * MT, end_block = (warp & (MT - 1)) * 16 < nrows ? first_block + MT : 0;  // (of a row tile without rows: none)
    const int at_row = (warp & (MT - 1)) * 16 + gid;  // of the tile's rows: this one and the eighth behind it
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    if (!ended) {
      uint32_t q[D / 16][4];
      int lo[2], hi[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row0 + at_row + 8 * i;
        const bool there = at_row + 8 * i < nrows;
        const int node = there ? r / G : 0, h = there ? r - node * G : 0;
        const bf16* src = (const bf16*)p.a.q + (size_t)(t.first + node) * p.a.q_stride + (size_t)(head * G + h) * D + tq * 2;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          q[k][i] = there ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16)) : 0u;
          q[k][2 + i] = there ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16 + 8)) : 0u;
        }
        const SharedWork::Row row = SharedWork::row(p.a, t, t.first + node);
        lo[i] = row.lo;
        hi[i] = row.hi;
      }
#pragma unroll 1
      for (int kt = t.kt_begin; kt < t.kt_end; ++kt, ++tile) {
        const int s = tile % FEW_STAGES, key0 = kt * BN;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (tile / FEW_STAGES) & 1));
        if (!ok) break;
        const uint32_t k_s = smem_u32(ring + s * 2 * KV_BYTES), v_s = k_s + KV_BYTES;
        const uint32_t bad = bad_pages[s];
        const bool ragged = bad != 0u || !SharedWork::whole(sh, t, key0);
        const Tile tl = {k_s, v_s, key0, bad, ragged};
        if (MT == 1)
          few_step<1>(tl, t, first_block, page_shift, scale, q, lo, hi, o, m, l);
        else
#pragma unroll 1
          for (int block = first_block; block < end_block; block += 2)
            few_step<2>(tl, t, block, page_shift, scale, q, lo, hi, o, m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
    }
    // Every working warp comes here once a share.  One whose wait ran out takes the others with it: no warp waits for one that
    // has left.
    const bool failed = any_warp(!ok);
    if (failed || ended) {
      if (failed && tid == 0) atomicOr(p.a.err, DSP_ERR_WAIT_LIMIT);
      return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // where a row of the tile is put down: a slot's row, or that of its sequence and head
    const int slot = t.slot;
    auto place = [&](int r) -> size_t {
      return slot >= 0 ? (size_t)slot * FEW_ROWS + r : SharedWork::row_part(sh, t, row0 + r);
    };
    float* out = slot >= 0 ? p.a.scratch.part_o : p.a.scratch.rows_o;
    float2* out_ml = reinterpret_cast<float2*>(slot >= 0 ? p.a.scratch.part_ml : p.a.scratch.rows_ml);
    if (MT == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = at_row + 8 * i;
        if (r >= nrows) continue;
        const size_t at = place(r);
        if (tq == 0) out_ml[at] = make_float2(m[i], l[i]);
        float* dst = out + at * D + tq * 2;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
      }
      continue;
    }
    const int r = tid >> 2;
    const bool mine = r < min(nrows, 16 * MT);
    const size_t at = place(mine ? r : 0);
    if (MT == 1)
      join_warps<1>(join, join_ml, o, m, l, mine ? out + at * D : nullptr, mine ? out_ml + at : nullptr);
    else
      join_warps<2>(join, join_ml, o, m, l, mine ? out + at * D : nullptr, mine ? out_ml + at : nullptr);
  }
}

// Launches the kernel; the arguments come checked.  Returns 0, or: 1 launch failed, 4 the shared-memory opt-in or the tensor maps
// failed.
int launch_shared_few(const DspSharedAttention& a, cudaStream_t stream) {
  const int page = a.page_size;
  FewParams p = {};
  p.a = a;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  CUtensorMap map_k, map_v, runs_k, runs_v;
  if (!make_map_pages(&map_k, a.k_pool, a.num_pages, a.sh.KVH, page, D, 1) ||
      !make_map_pages(&map_v, a.v_pool, a.num_pages, a.sh.KVH, page, D, 1))
    return 4;
  // a pool of fewer pages than a key tile has gives no map of runs
  p.page_runs = make_map_pages(&runs_k, a.k_pool, a.num_pages, a.sh.KVH, page, D, BN / page) &&
                make_map_pages(&runs_v, a.v_pool, a.num_pages, a.sh.KVH, page, D, BN / page);
  if (!p.page_runs) {
    runs_k = map_k;
    runs_v = map_v;
  }
  static bool allowed[MAX_DEVICES] = {};  // asked for once a device
  const int device = current_device();
  if (device < 0 || !allowed[device]) {
    if (cudaFuncSetAttribute(shared_attn_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM) != cudaSuccess) return 4;
    if (device >= 0) allowed[device] = true;
  }
  return launch_pdl(shared_attn_few_kernel, dim3((unsigned)a.ctas), dim3(FEW_THREADS), (size_t)FEW_SMEM, stream, p, map_k, map_v, runs_k,
                    runs_v) == cudaSuccess
             ? 0
             : 1;
}
}  // namespace
