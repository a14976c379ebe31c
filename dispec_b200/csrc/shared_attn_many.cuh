// Attention of shared beginnings that many rows see, on the fifth-generation tensor cores: bfloat16 in, 32-bit softmax and
// accumulation (the formula: shared_attn.cu; how the work is cut: shared_schedule.cuh).  Compiled once per head size
// (-DDSP_HEAD_DIM=64 or 128).
//
// One CTA an SM walks its run of units.  A share is up to 256 query rows of one key/value head, two tiles of 128, over key tiles of
// 64: both row tiles use a key tile while it is in shared memory.  S = Q K^T and O += P V are tcgen05.mma with S and O in tensor
// memory (all of its 512 columns in heads of 128); each row tile has two score buffers, and the weights P take the place of the scores
// that they were formed from, so that the scores of the next tile are there when a tile's softmax ends.  Roles:
//   warp 0      requests the key and value tiles, which share a ring that runs on from share to share;
//   warps 1, 2  issue the products of a row tile each: O += P V of key tile j, then S of tile j + 2 into the same buffer, which the
//               pipe does in that order (one warp for both took 1,000 cycles to issue the twelve products of a step, and then those
//               of the other row tile);
//   warps 4..11 two softmax groups of four warps, one for each row tile; thread r of a group owns row r.  They bring the queries
//               into shared memory, and store a share's rows while the next one's first scores are being formed.
// What bounds it: the softmax, 2,050 cycles for both row tiles' 256 rows and a key tile, of which the products are 1,000: 64
// sequences of 40 heads of 128 on 8 (320 rows) behind 32,768 tokens: 76 us, 0.57 PFLOP/s with the rows there are, 1.8 TB/s.  Other cuts
// of the same work, for the whole call where this one took 116 us (107 since the other kernel begins beside it): one issuing warp for both row tiles 141, key tiles of 128 119, two threads a row (a meeting
// a tile: 2,400 cycles) 122, one row tile a CTA whose two groups take key tiles in turn 130 (each tile is then requested twice as
// often, eight requests of scattered pages).
// Nothing but barriers in memory joins the roles; every wait is bounded, and one that runs out sets the device error word.
// Value rows that no row of the item may see are zeroed in shared memory before the output product, and so are, in tiles that
// not every row sees whole, values that are not finite, which a weight of 0 would carry to rows that do not see them: behind the
// product they are added to the rows that do.
#pragma once
#include "rows_attn_tcgen05.cuh"
#include "shared_schedule.cuh"

namespace {
constexpr int MANY_THREADS = 384;
constexpr int MANY_ROWS = 1 << ROW_SHIFT_MANY;
static_assert(MANY_ROWS == 2 * BM, "two row tiles");
constexpr int Q_BYTES = BM / 8 * GROUP;
constexpr int MANY_STAGES = 8;  // key and value tiles in turn
static_assert(MANY_STAGES % 2 == 0, "a tile's keys and values lie in neighbouring stages");
constexpr int MANY_SMEM = 2 * Q_BYTES + MANY_STAGES * KV_BYTES + 1024;
constexpr int MANY_O_COL = 4 * BN;  // tensor memory: two score buffers of each row tile, then the accumulators
static_assert(MANY_O_COL + 2 * D <= TMEM_COLS, "tensor memory layout");
constexpr int KNOWN = 8;                        // shares that are told ahead

__global__ void __launch_bounds__(MANY_THREADS, 1)
shared_attn_many_kernel(const __grid_constant__ Params<SharedWork> p, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap runs_k,
                        const __grid_constant__ CUtensorMap runs_v) {
  typedef shared::Share Share;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* q_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* ring = q_s + 2 * Q_BYTES;
  __shared__ __align__(8) uint64_t full[MANY_STAGES], empty[MANY_STAGES];  // landed; every product with it is complete
  __shared__ __align__(8) uint64_t q_full[2];          // the queries of a row tile are in shared memory
  // of row tile g and key tiles of one parity: scores complete; weights written; output product complete
  __shared__ __align__(8) uint64_t s_full[2][2], p_full[2][2], o_done[2][2];
  // Of a tile that is not seen whole, n, in n % 8: one group has cleaned the values for both.  (Those of tile n + 8 land when the
  // products of tile n + 4 are complete.)
  __shared__ __align__(8) uint64_t cleaned[8];
  __shared__ __align__(8) uint64_t known[KNOWN], left[KNOWN];  // a share is told; the warps that go by it have left it
  __shared__ Share shares[KNOWN];                  // share k in k % KNOWN, told before its first tile is requested
  // Of key tile n, in n % 16; bit j: page j is not there.  Keys of tile n + 6 are asked for when the scores of tile n + 2 are complete,
  // whose buffer the softmax of tile n has left.
  __shared__ uint32_t bad_pages[16];
  static_assert(MANY_STAGES / 2 + 2 < 16, "tiles that may be looked at");
  __shared__ int odd_share[KNOWN];  // share k in k % KNOWN: numbers were taken out of its values (one group may be a share ahead)
  __shared__ uint32_t tmem_slot;
  __shared__ shared::Plan plan;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const shared::Shape& sh = p.a.sh;
  const int G = sh.G;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tid == 64) {
    for (int s = 0; s < MANY_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&q_full[g], 4);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s_full[g][b], 1);
        mbar_init(&p_full[g][b], 4);
        mbar_init(&o_done[g][b], 1);
      }
    }
    for (int k = 0; k < KNOWN; ++k) {
      mbar_init(&known[k], 1);
      mbar_init(&left[k], 10);  // the warps of the products and the softmax warps
      mbar_init(&cleaned[k], 4);
    }
    for (int k = 0; k < KNOWN; ++k) odd_share[k] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();  // (the other kernel's CTAs begin where these end, and do not wait for them)
  shared::make_plan(sh, plan.groups, plan.run, blockIdx.x, gridDim.x);  // (meets)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  const int page_size = p.a.page_size, page_shift = __ffs(page_size) - 1;
  bool ok = true;

  if (warp == 0) {
    // ---- requests
    shared::Walk w;
    bool more = w.begin(sh, plan.run, blockIdx.x);
    const int pages_per_tile = BN >> page_shift, ppt_shift = 6 - page_shift, chunk_tiles = 32 >> ppt_shift;
    const int page_in_tile = lane & (pages_per_tile - 1);
    const uint32_t tile_lanes = (1u << pages_per_tile) - 1u;  // (at most eight pages)
    const uint32_t page_bytes = (uint32_t)page_size * D * 2;
    // ids of the pages of 32 / pages_per_tile tiles from tile kt on, lane by lane (-2: not wanted)
    auto load_chunk = [&](const Share& t, int kt) -> int {
      const int of = kt + (lane >> ppt_shift), first = of * BN + page_in_tile * page_size;
      if (of >= t.kt_end || first >= t.end || first + page_size <= t.begin) return -2;
      const int j = first >> page_shift;
      return j < p.a.table_width ? max(p.a.page_table[(size_t)t.seq * p.a.pt_stride + j], -1) : -1;
    };
    int share = 0, tile = 0, pg_first = more ? load_chunk(w.at, w.at.kt_begin) : -2;
    while (more && ok) {
      const Share t = w.at;
      ok = __all_sync(0xffffffffu, share < KNOWN || mbar_wait(&left[share % KNOWN], (share / KNOWN - 1) & 1));
      if (!ok) break;
      if (lane == 0) {
        shares[share % KNOWN] = t;
        mbar_arrive(&known[share % KNOWN]);
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
          const bool bad = pg == -1 || pg >= p.a.num_pages;  // recorded, not loaded, its keys are hidden
          if (bad) {
            atomicOr(p.a.err, DSP_ERR_BAD_PAGE);
            pg = -1;
          }
          bad_mask = __ballot_sync(0xffffffffu, bad);
          live_mask = __ballot_sync(0xffffffffu, pg >= 0);
          const int first_pg = __shfl_sync(0xffffffffu, pg, lane & ~(pages_per_tile - 1));
          run_mask = __ballot_sync(0xffffffffu, pg >= 0 && pg == first_pg + page_in_tile && first_pg + pages_per_tile <= p.a.num_pages);
        }
        const int shift = in_chunk << ppt_shift;
        const uint32_t live = (live_mask >> shift) & tile_lanes;
        const bool in_run = p.page_runs && ((run_mask >> shift) & tile_lanes) == tile_lanes;
        const bool mine = lane >> ppt_shift == in_chunk;
        const int s = 2 * tile % MANY_STAGES, use = 2 * tile / MANY_STAGES, groups = page_size >> 3, dst = page_in_tile * groups * GROUP;
#pragma unroll 1
        for (int v = 0; v < 2 && ok; ++v) {
          ok = __all_sync(0xffffffffu, use == 0 || mbar_wait(&empty[s + v], (use - 1) & 1));
          if (!ok) break;
          if (lane == 0) {
            if (v == 0) bad_pages[tile & 15] = (bad_mask >> shift) & tile_lanes;  // published by the arrival
            if (live == 0)
              mbar_arrive(&full[s + v]);
            else
              mbar_expect_tx(&full[s + v], (uint32_t)__popc(live) * page_bytes);
          }
          __syncwarp();
          unsigned char* at = ring + (s + v) * KV_BYTES;
          if (mine && in_run) {
            if (page_in_tile == 0) load_pages(at, v ? &runs_v : &runs_k, &full[s + v], t.head * groups, pg);
          } else if (mine && pg >= 0) {
            load_pages(at + dst, v ? &map_v : &map_k, &full[s + v], t.head * groups, pg);
          }
        }
        if (!ok) break;
      }
      ++share;
    }
    ok = __all_sync(0xffffffffu, ok && (share < KNOWN || mbar_wait(&left[share % KNOWN], (share / KNOWN - 1) & 1)));
    if (lane == 0 && ok) {  // the end
      shares[share % KNOWN].seq = -1;
      mbar_arrive(&known[share % KNOWN]);
    }
  } else if (warp <= 2) {
    // ---- products of row tile g
    const int g = warp - 1;
    const uint32_t idesc_s = umma_idesc(BM, BN), idesc_o = umma_idesc(BM, D) | (1u << 16);  // B (values) is N-major
    const uint64_t q_desc = key_desc(smem_u32(q_s + g * Q_BYTES), GROUP);
    const uint64_t k_desc0 = key_desc(smem_u32(ring), GROUP), v_desc0 = value_desc(smem_u32(ring), GROUP);
    const uint32_t s_cols = tmem_base + (uint32_t)(2 * g * BN), o_cols = tmem_base + (uint32_t)(MANY_O_COL + g * D);
    const bool leader = elect_one();
    int tile = 0, uses[2] = {0, 0};  // key tiles; of the score buffers
    uint32_t q_uses = 0, clean_uses = 0;  // bit n % 8: parity of cleaned[n % 8]
    auto landed = [&](int of, int v) { return __all_sync(0xffffffffu, mbar_wait(&full[(2 * of + v) % MANY_STAGES], (2 * of / MANY_STAGES) & 1)); };
    auto scores = [&](int of, int b) {  // over the keys in the ring's place for that tile, into buffer b; then the keys may go
      const int s = 2 * of % MANY_STAGES;
      if (leader) {
        const uint64_t k_desc = k_desc0 + (uint64_t)(s * (KV_BYTES >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = (uint64_t)(((uint32_t)(k >> 2) * SLICE + (uint32_t)(k & 3) * 32u) >> 4);
          umma(s_cols + (uint32_t)(b * BN), q_desc + off, k_desc + off, idesc_s, k != 0);
        }
        umma_commit(&s_full[g][b]);
        umma_commit(&empty[s]);
      }
      __syncwarp();
    };
#pragma unroll 1
    for (int share = 0; ok; ++share) {
      ok = __all_sync(0xffffffffu, mbar_wait(&known[share % KNOWN], (share / KNOWN) & 1));
      if (!ok) break;
      const Share& t = shares[share % KNOWN];
      if (t.seq < 0) break;
      const int tiles = t.kt_end - t.kt_begin, kt_begin = t.kt_begin;
      if (t.n * G - t.row_tile * MANY_ROWS <= g * BM) {
        // no rows of this tile: keys and values may go as they come
#pragma unroll 1
        for (int j = 0; j < tiles && ok; ++j, ++tile)
#pragma unroll 1
          for (int v = 0; v < 2 && ok; ++v) {
            ok = landed(tile, v);
            if (v == 1 && ok && (bad_pages[tile & 15] != 0u || !SharedWork::whole(sh, t, (kt_begin + j) * BN))) clean_uses ^= 1u << (tile & 7);
            if (lane == 0 && ok) mbar_arrive(&empty[(2 * tile + v) % MANY_STAGES]);
          }
        if (lane == 0) mbar_arrive(&left[share % KNOWN]);
        continue;
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&q_full[g], q_uses++ & 1));
      tc_fence_after();
#pragma unroll 1
      for (int j = 0; j < min(tiles, 2) && ok; ++j) {
        ok = landed(tile + j, 0);
        if (ok) scores(tile + j, j);
      }
#pragma unroll 1
      for (int j = 0; j < tiles && ok; ++j, ++tile) {
        const bool another = j + 2 < tiles;
        const int b = j & 1, sv = (2 * tile + 1) % MANY_STAGES;
        ok = landed(tile, 1);
        if (!ok) break;
        if (bad_pages[tile & 15] != 0u || !SharedWork::whole(sh, t, (kt_begin + j) * BN)) {
          ok = __all_sync(0xffffffffu, mbar_wait(&cleaned[tile & 7], (clean_uses >> (tile & 7)) & 1));
          clean_uses ^= 1u << (tile & 7);
          if (!ok) break;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&p_full[g][b], (b ? uses[1] : uses[0]) & 1));
        if (!ok) break;
        if (b)
          ++uses[1];
        else
          ++uses[0];
        tc_fence_after();
        if (leader) {
          const uint64_t v_desc = v_desc0 + (uint64_t)(sv * (KV_BYTES >> 4));
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            umma_a_tmem(o_cols, s_cols + (uint32_t)(b * BN + k * 8), v_desc + (uint64_t)(k * (2 * GROUP >> 4)), idesc_o, j != 0 || k != 0);
          umma_commit(&o_done[g][b]);
          umma_commit(&empty[sv]);
        }
        __syncwarp();
        if (another) {
          ok = landed(tile + 2, 0);
          if (ok) scores(tile + 2, b);
        }
      }
      if (lane == 0) mbar_arrive(&left[share % KNOWN]);
    }
  } else if (warp >= 4) {
    // ---- softmax
    const int g = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane, r4 = r & ~3;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr0 = lane_addr + (uint32_t)(2 * g * BN), o_addr = lane_addr + (uint32_t)(MANY_O_COL + g * D);
    const float scale = p.scale_log2;
    // thread r brings row r of the group's tile of a share's queries (rows past the item are zero)
    auto bring_queries = [&](const Share& t) {
      const int rr = t.row_tile * MANY_ROWS + g * BM + r, node = rr / G;
      const bool there = rr < t.n * G;
      const bf16* src = (const bf16*)p.a.q + (size_t)(t.first + (there ? node : 0)) * p.a.q_stride + (size_t)(t.head * G + (there ? rr - node * G : 0)) * D;
      const uint32_t dst = smem_u32(q_s + g * Q_BYTES) + (uint32_t)(r >> 3) * GROUP + (uint32_t)(r & 7) * 128u;
#pragma unroll
      for (int c0 = 0; c0 < D / 8; c0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = there ? __ldg(reinterpret_cast<const uint4*>(src) + c0 + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 8; ++c) st_shared16(dst + (uint32_t)(c0 >> 3) * SLICE + (uint32_t)((c ^ (r & 7)) << 4), x[c]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[g]);
    };
    auto has_rows = [&](const Share& t) { return t.n * G - t.row_tile * MANY_ROWS > g * BM; };
    int tile = 0, uses[2] = {0, 0};  // key tiles; of this group, by parity in the share
    bool brought = false;
#pragma unroll 1
    for (int share = 0; ok; ++share) {
      ok = __all_sync(0xffffffffu, mbar_wait(&known[share % KNOWN], (share / KNOWN) & 1));
      if (!ok) break;
      const Share& t = shares[share % KNOWN];
      if (t.seq < 0) break;
      const int tiles = t.kt_end - t.kt_begin;
      if (!has_rows(t)) {
        tile += tiles;
        __syncwarp();
        if (lane == 0) mbar_arrive(&left[share % KNOWN]);
        continue;
      }
      if (!brought) bring_queries(t);
      brought = false;
      const int row0 = t.row_tile * MANY_ROWS + g * BM, nrows = min(BM, t.n * G - row0);
      const bool row_ok = r < nrows, warp_ok = quarter * 32 < nrows;  // a warp without rows only keeps the barriers going
      const bool alone = t.n * G - t.row_tile * MANY_ROWS <= BM;      // the other group has no rows
      const int node = t.first + (row_ok ? (row0 + r) / G : 0);
      float m_run = -INFINITY, l_run = 0.f;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j, ++tile) {
        const int key0 = (t.kt_begin + j) * BN, b01 = j & 1;
        const uint32_t s_addr = s_addr0 + (uint32_t)(b01 * BN);
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[g][b01], (b01 ? uses[1] : uses[0]) & 1));
        if (!ok) break;
        tc_fence_after();
        // (the tile's keys have landed, and with them what was put down of its pages)
        const uint32_t bad = bad_pages[tile & 15];
        const bool ragged = bad != 0u || !SharedWork::whole(sh, t, key0);
        if (warp_ok) {
          uint32_t a[32], b[32];
          tmem_ld32_nowait(s_addr, a);
          tmem_ld32_nowait(s_addr + 32, b);
          unsigned long long seen = ~0ull;
          if (ragged) {
            seen = row_ok ? SharedWork::seen_keys(p.a, t, SharedWork::row(p.a, t, node), key0) : 0ull;
#pragma unroll 1
            for (int k = 0; k < BN >> page_shift; ++k)
              if ((bad >> k) & 1u) seen &= ~((page_size == 64 ? ~0ull : (1ull << page_size) - 1ull) << (k << page_shift));
          }
          tmem_ld_wait();
          if (ragged) {
            const uint32_t lo = (uint32_t)seen, hi = (uint32_t)(seen >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              a[c] = (lo >> c) & 1u ? a[c] : 0xff800000u;  // -inf
              b[c] = (hi >> c) & 1u ? b[c] : 0xff800000u;
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
          const float2 scale2 = make_float2(scale, scale), neg_m2 = make_float2(neg_m, neg_m);
          float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(a[c]), __uint_as_float(a[c + 1])), scale2, neg_m2);
            const float2 y = fma2(make_float2(__uint_as_float(b[c]), __uint_as_float(b[c + 1])), scale2, neg_m2);
            const float2 ex = make_float2(ex2(x.x), ex2(x.y));
            const float2 ey = c / 2 % 4 < EX2_FMA ? ex2_fma(y) : make_float2(ex2(y.x), ex2(y.y));
            // the second product takes weights of eight bits, as it takes values (their sum is of the 32-bit ones)
            sum0 = add2(sum0, ex);
            sum1 = add2(sum1, ey);
            pk[c / 2] = pack2(ex.x, ex.y);
            pk[16 + c / 2] = pack2(ey.x, ey.y);
          }
          sum0 = add2(sum0, sum1);
          l_run = l_run * alpha + (sum0.x + sum0.y);
          __syncwarp();
          tmem_st32(s_addr, pk);  // over the scores
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            // the product before this tile's has to be complete (this tile's waits for these weights)
            ok = __all_sync(0xffffffffu, mbar_wait(&o_done[g][b01 ^ 1], ((b01 ? uses[0] : uses[1]) - 1) & 1));
            if (!ok) break;
            tc_fence_after();
            rescale(o_addr, alpha);
          }
        }
        // values that 0 as a weight would not keep out
        if (ragged && (alone || (tile & 1) == g)) {
          const int sv = (2 * tile + 1) % MANY_STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait(&full[sv], (2 * tile / MANY_STAGES) & 1));
          if (!ok) break;
          if (clean_values<SharedWork>(p, t, smem_u32(ring + sv * KV_BYTES), t.kt_begin + j, bad, r)) odd_share[share % KNOWN] = share;
          __syncwarp();
          if (lane == 0) mbar_arrive(&cleaned[tile & 7]);
        }
        __syncwarp();
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g][b01]);
        if (b01)
          ++uses[1];
        else
          ++uses[0];
      }
      if (!ok) break;
      // the next share's queries take the place of this one's, whose scores are all there; where it is not known yet, they are
      // brought when it is
      const bool known_ahead = mbar_wait_limit(&known[(share + 1) % KNOWN], ((share + 1) / KNOWN) & 1, 1);
      if (__all_sync(0xffffffffu, known_ahead)) {
        const Share& next = shares[(share + 1) % KNOWN];
        if (next.seq >= 0 && has_rows(next)) {
          bring_queries(next);
          brought = true;
        }
      }
      {
        const int b01 = (tiles - 1) & 1;  // of the last tile, whose product is behind all others
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done[g][b01], ((b01 ? uses[1] : uses[0]) - 1) & 1));
      }
      if (!ok) break;
      tc_fence_after();
      if (odd_share[share % KNOWN] == share && warp_ok) {
        add_odd_values<SharedWork>(p, t, 0, 1, SharedWork::row(p.a, t, node), row_ok, o_addr);
        __syncwarp();
      }
      // the rows' sums, four neighbouring lanes together 64 bytes of each of their rows
      if (warp_ok) {
        const int slot = t.slot;
        auto place = [&](int k) -> size_t {  // of the tile's row k
          return slot >= 0 ? (size_t)slot * MANY_ROWS + g * BM + k : SharedWork::row_part(sh, t, row0 + k);
        };
        size_t at[4];
        const int n4 = min(4, nrows - r4);
#pragma unroll
        for (int k = 0; k < 4; ++k) at[k] = place(k < n4 ? r4 + k : 0);
        float* out = (slot >= 0 ? p.a.scratch.part_o : p.a.scratch.rows_o) + (lane & 3) * 4;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t ov[32];
          __syncwarp();
          tmem_ld32(o_addr + (uint32_t)c0, ov);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 x[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = make_uint4(ov[16 * h + 4 * c], ov[16 * h + 4 * c + 1], ov[16 * h + 4 * c + 2], ov[16 * h + 4 * c + 3]);
            transpose4(x);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (k < n4) *reinterpret_cast<uint4*>(out + at[k] * D + c0 + 16 * h) = x[k];
          }
        }
        if (row_ok) reinterpret_cast<float2*>(slot >= 0 ? p.a.scratch.part_ml : p.a.scratch.rows_ml)[place(r)] = make_float2(m_run, l_run);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&left[share % KNOWN]);
    }
  }
  if (!ok && lane == 0) atomicOr(p.a.err, DSP_ERR_WAIT_LIMIT);
  if (__syncthreads_or(!ok)) {
    // let copies and products that are still on their way land before the shared memory goes away
#pragma unroll 1
    for (int i = 0; i < 2000; ++i) __nanosleep(100);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}

// Launches the kernel; the arguments come checked.  Returns 0, or: 1 launch failed, 4 the shared-memory opt-in or the tensor maps
// failed.
int launch_shared_many(const DspSharedAttention& a, cudaStream_t stream) {
  const int page = a.page_size;
  Params<SharedWork> p = {};
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
    if (cudaFuncSetAttribute(shared_attn_many_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MANY_SMEM) != cudaSuccess) return 4;
    if (device >= 0) allowed[device] = true;
  }
  return launch_pdl(shared_attn_many_kernel, dim3((unsigned)a.ctas), dim3(MANY_THREADS), (size_t)MANY_SMEM, stream, p, map_k, map_v,
                    runs_k, runs_v) == cudaSuccess
             ? 0
             : 1;
}
}  // namespace
