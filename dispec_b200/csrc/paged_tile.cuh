// A tile of 64 keys of one head in shared memory, as TMA brings its pages (make_map_pages in tcgen05_common.cuh), for kernels that are
// compiled per head size (-DDSP_HEAD_DIM): [group of 8 keys][slice of 64 columns][8 rows of 128 bytes], a page's rows in one
// request.  Heads of 32 have one slice of 32 columns, rows of 64 bytes and a swizzle of 64.
#pragma once
#include "rows_schedule.cuh"
#include "tcgen05_common.cuh"

#ifndef DSP_HEAD_DIM
#error "compile with -DDSP_HEAD_DIM=<head size>"
#endif
#define DSP_CAT2(a, b) a##b
#define DSP_CAT(a, b) DSP_CAT2(a, b)

namespace {
using namespace tc;

constexpr int D = DSP_HEAD_DIM;
static_assert(D == 32 || D == 64 || D == 128, "head sizes with such tiles");
constexpr int BN = KEYS_PER_TILE;
constexpr int SLICE_COLS = D < 64 ? D : 64, KD = D / SLICE_COLS;
constexpr int ROW_BYTES = SLICE_COLS * 2, SLICE = 8 * ROW_BYTES;
static_assert(D == 32 || SLICE == KEY_SLICE, "as the tensor maps have it");
constexpr int GROUP = KD * SLICE;
constexpr int KV_BYTES = BN / 8 * GROUP;
constexpr float RESCALE_STEP = 8.f;  // the running maximum of a softmax follows the true one in steps of 2^8

// Where a row's 16-byte piece lies, from the row's beginning on; `in_group`: the row's place in its group of 8.
__device__ __forceinline__ uint32_t piece_at(int piece, int in_group) {
  if constexpr (D == 32)
    return (uint32_t)(piece ^ (in_group >> 1)) << 4;
  else
    return (uint32_t)(piece >> 3) * SLICE + ((uint32_t)((piece & 7) ^ in_group) << 4);
}
// ... and a row of its tile.
__device__ __forceinline__ uint32_t row_at(int row) { return (uint32_t)(row >> 3) * GROUP + (uint32_t)(row & 7) * ROW_BYTES; }

// Two bfloat16 values: one that is not finite; the same with 0 in its place.
__device__ __forceinline__ bool has_odd(uint32_t x) { return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t without_odd(uint32_t x) {
  return ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u);
}
}  // namespace
