// What the kernels over rows of queries and their schedules (tree_schedule.cuh, shared_schedule.cuh) have in common.
#pragma once
#include "common.cuh"

// Sizes of tiles are powers of two, and shifts: a CTA runs the search for its run once, and fetches every instruction of a division
// for it.
constexpr int KEY_SHIFT = 6, KEYS_PER_TILE = 1 << KEY_SHIFT;
constexpr int ROW_SHIFT_TENSOR_CORES = 7;  // 128 rows a tile of the tensor-core kernel
constexpr int ROW_SHIFT_MANY = 8;          // 256 of the one for shared beginnings that many rows see
constexpr int ROW_SHIFT_FEW = 6;           // 64 of the one for sequences whose keys few rows see
constexpr int ROW_SHIFT_32BIT = 5;         // 32 of the 32-bit kernel

struct NoPlan {};  // a schedule whose CTAs find their runs without working anything out together

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
