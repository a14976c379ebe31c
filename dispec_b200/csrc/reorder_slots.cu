// Slots of pools follow a choice: in every pool [layers, slots, ...]
//     pool[:, dst[i]] = pool[:, src[i]]   for all i, as though all were read before any is written.
//
// Bytes of different columns have nothing to do with each other.  So a block takes some columns of one layer of one pool for
// ALL i: it holds them in shared memory or in registers, meets, and writes them.  A slot may be read by several and
// written by another in one call, in place and without a copy of anything, and no block waits for another.
//
// Memory bounds it: 906 MB in rows of 32 KB (48 layers of keys and values, read and written) take 136 us, 151 MB in rows of 512 KB
// (12 layers of states) 23.6: 6.6 and 6.4 TB/s.
//
// The next kernel does not begin before the last block has left: what is written here are stored keys and values too, which the
// attention of single tokens reads in front of its wait.
//
// dst ascends, so that no slot is written twice; what does not ascend, or names a slot that is not there, is left from there on
// and recorded.
#include "tcgen05_common.cuh"
#include "tensor_checks.cuh"

namespace {
constexpr int MAX_POOLS = 64, EACH = 8;

struct Pool {
  char* data;
  long row_bytes;  // of a slot in one layer
  int slots, first_block;
  int chunks;      // blocks of a layer
};
struct Args {
  Pool pools[MAX_POOLS];
  const int *src, *dst;
  int count, pools_n;
  int chunk_shift, chunk_bytes;  // of an entry in a block: 1 << chunk_shift pieces; of bulk copies
  int* err;
};

// The pool of a block: the last one whose first block is not behind it.
__device__ __forceinline__ const Pool& pool_of(const Args& a) {
  int p = 0;
  for (int step = MAX_POOLS / 2; step > 0; step >>= 1)
    if (p + step < a.pools_n && a.pools[p + step].first_block <= (int)blockIdx.x) p += step;
  return a.pools[p];
}
// How many entries are copied, by the whole block.
__device__ __forceinline__ int sound_entries(const Args& a, const Pool& pool, int* bad) {
  if (threadIdx.x == 0) *bad = a.count;
  __syncthreads();
  for (int i = threadIdx.x; i < a.count; i += blockDim.x) {
    const int s = a.src[i], d = a.dst[i], before = i > 0 ? a.dst[i - 1] : -1;
    if (s < 0 || s >= pool.slots || d < 0 || d >= pool.slots || d <= before) atomicMin(bad, i);
  }
  __syncthreads();
  if (*bad < a.count && threadIdx.x == 0) atomicOr(a.err, DSP_ERR_BAD_GROUP);
  return *bad;
}

// Rows of whole 16-byte pieces and up to BULK_ENTRIES entries: the columns of an entry are one bulk copy into shared memory and one
// back, of whole lines of 128 bytes where six blocks an SM hold them, else of 96 bytes at least.  The two calls above: 136 and 23.6 us; with
// 48 KB a block and copies of 336 and 4,096 bytes 160 and 24.9; lines, and room for 48 KB all the same (four blocks an SM) 165; lines with
// 74 KB 140 and 25.3.  Through registers, eight pieces a thread, 203 and 32.7; more entries, and rows of other sizes, go that way
// (rows of 32 KB in 24 layers, behind a flushed L2: 512 entries 3.4 TB/s, 513 3.0; rows of 32,776 bytes 2.1).
constexpr int BULK_THREADS = 128, BULK_ENTRIES = 512, BULK_BYTES = 48 * 1024, LINE_BYTES = 37 * 1024;
__global__ void __launch_bounds__(BULK_THREADS)
reorder_bulk_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(128) unsigned char stage[];
  __shared__ int bad;
  __shared__ __align__(8) uint64_t landed;
  const int tid = threadIdx.x;
  const Pool& pool = pool_of(a);
  const int block = blockIdx.x - pool.first_block, layer = block / pool.chunks, chunk = block - layer * pool.chunks;
  const long column = (long)chunk * a.chunk_bytes;
  const uint32_t bytes = (uint32_t)min((long)a.chunk_bytes, pool.row_bytes - column);
  char* base = pool.data + (size_t)layer * pool.slots * pool.row_bytes + column;
  if (tid == 0) {
    tc::mbar_init(&landed, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  const int count = sound_entries(a, pool, &bad);
  if (count == 0) return;
  if (tid == 0) tc::mbar_expect_tx(&landed, bytes * (uint32_t)count);
  __syncthreads();
  for (int i = tid; i < count; i += BULK_THREADS)
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     tc::smem_u32(stage + (size_t)i * a.chunk_bytes)),
                 "l"(base + (size_t)a.src[i] * pool.row_bytes), "r"(bytes), "r"(tc::smem_u32(&landed))
                 : "memory");
  if (!tc::mbar_wait(&landed, 0)) {
    atomicOr(a.err, DSP_ERR_WAIT_LIMIT);
    // let copies that are still on their way land before the shared memory goes away
#pragma unroll 1
    for (int i = 0; i < 2000; ++i) __nanosleep(100);
    return;
  }
  for (int i = tid; i < count; i += BULK_THREADS)
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(base + (size_t)a.dst[i] * pool.row_bytes),
                 "r"(tc::smem_u32(stage + (size_t)i * a.chunk_bytes)), "r"(bytes)
                 : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

template <typename Piece, int THREADS>
__global__ void __launch_bounds__(THREADS)
reorder_kernel(const __grid_constant__ Args a) {
  __shared__ int bad;
  const int tid = threadIdx.x;
  const Pool& pool = pool_of(a);
  const int block = blockIdx.x - pool.first_block, layer = block / pool.chunks, chunk = block - layer * pool.chunks;
  pdl_wait();
  const int count = sound_entries(a, pool, &bad);
  const long in_row = pool.row_bytes / (long)sizeof(Piece);
  Piece* base = reinterpret_cast<Piece*>(pool.data) + (size_t)layer * pool.slots * in_row;
  const long column0 = (long)chunk << a.chunk_shift;
  const int mask = (1 << a.chunk_shift) - 1;
  Piece x[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int q = tid + k * THREADS, i = q >> a.chunk_shift;
    const long column = column0 + (q & mask);
    if (i < count && column < in_row) x[k] = base[(size_t)a.src[i] * in_row + column];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int q = tid + k * THREADS, i = q >> a.chunk_shift;
    const long column = column0 + (q & mask);
    if (i < count && column < in_row) base[(size_t)a.dst[i] * in_row + column] = x[k];
  }
}
}  // namespace

// tensors: src, dst, pools ...
extern "C" int dsp_reorder_slots(const DspTensor* t, long pools, cudaStream_t stream) {
  const DspTensor &src = t[0], &dst = t[1];
#define REORDER_REQUIRE(cond, ...) DSP_REQUIRE(cond, "reorder_slots: " __VA_ARGS__)
  REORDER_REQUIRE(src.device >= 0, "CUDA tensors only (there is no CPU path)");
  REORDER_REQUIRE(pools >= 1 && pools <= MAX_POOLS, "%ld pools, 1 to %d expected", pools, MAX_POOLS);
  REORDER_REQUIRE(src.dims == 1, "src must be one-dimensional");
  const long n = src.size[0];
  REORDER_REQUIRE(tensor_is(src, DSP_T_I32, src.device, 1, n) && tensor_is(dst, DSP_T_I32, src.device, 1, n),
                  "src and dst must be contiguous int32 of one length on one device");
  Args a = {};
  uintptr_t bits = 0, ends[MAX_POOLS];
  const DspTensor& first = t[2];
  for (long p = 0; p < pools; ++p) {
    const DspTensor& x = t[2 + p];
    REORDER_REQUIRE(x.dims >= 3 && x.dims <= DSP_T_DIMS && x.contiguous && x.device == src.device && x.dtype != DSP_T_OTHER,
                    "pool %ld must be a contiguous tensor [layers, slots, ...] of three to five dimensions, float32, bfloat16, int32 or int64, on the device of src", p);
    REORDER_REQUIRE(x.size[1] == first.size[1], "pool %ld has %ld slots, the first one %ld", p, x.size[1], first.size[1]);
    long elements = 1;
    for (int k = 2; k < x.dims; ++k) elements *= x.size[k];
    a.pools[p].data = (char*)x.data;
    a.pools[p].row_bytes = elements * (x.dtype == DSP_T_BF16 ? 2 : x.dtype == DSP_T_I64 ? 8 : 4);
    a.pools[p].slots = (int)x.size[1];
    REORDER_REQUIRE(x.size[1] <= 0x7fffffff, "pool %ld has too many slots", p);
    bits |= (uintptr_t)x.data | (uintptr_t)a.pools[p].row_bytes;
    const uintptr_t at = (uintptr_t)x.data;
    ends[p] = at + (uintptr_t)(x.size[0] * x.size[1] * a.pools[p].row_bytes);
    for (long o = 0; o < p; ++o)
      REORDER_REQUIRE(at >= ends[o] || ends[p] <= (uintptr_t)a.pools[o].data, "pools %ld and %ld have parts of the same memory", o, p);
  }
  if (n == 0) return 0;
  // the widest pieces that all rows consist of; as much of an entry in a block as it can hold
  const long piece = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
  const bool bulk = piece == 16 && n <= BULK_ENTRIES;
  const int threads = n <= 512 ? 256 : 1024;  // (rows of 64 bytes at least up to 2,048 entries)
  REORDER_REQUIRE(n <= (long)threads * EACH, "%ld slots to be copied, at most %d", n, 1024 * EACH);
  while ((n << (a.chunk_shift + 1)) <= (long)threads * EACH) ++a.chunk_shift;
  const long chunk_bytes = bulk ? (n * 128 <= LINE_BYTES ? LINE_BYTES / n / 128 * 128 : BULK_BYTES / n / 16 * 16) : piece << a.chunk_shift;
  a.chunk_bytes = (int)chunk_bytes;
  long blocks = 0;
  for (long p = 0; p < pools; ++p) {
    Pool& x = a.pools[p];
    const long chunks = (x.row_bytes + chunk_bytes - 1) / chunk_bytes;
    x.chunks = (int)max(chunks, 1L);
    x.first_block = (int)blocks;
    blocks += chunks * t[2 + p].size[0];
    REORDER_REQUIRE(blocks <= 0x7fffffff && chunks <= 0x7fffffff, "the pools are too large for one call");
  }
  if (blocks == 0) return 0;
  REORDER_REQUIRE(current_device() == src.device, "the tensors are on device %d, the current device is %d", src.device, current_device());
  // (blocks read the lists while others write)
  for (const DspTensor* list : {&src, &dst})
    for (long p = 0; p < pools; ++p)
      REORDER_REQUIRE((uintptr_t)list->data >= ends[p] || (uintptr_t)list->data + 4 * (uintptr_t)n <= (uintptr_t)a.pools[p].data,
                      "src or dst lies in pool %ld", p);
  a.src = (const int*)src.data;
  a.dst = (const int*)dst.data;
  a.count = (int)n;
  a.pools_n = (int)pools;
  a.err = dsp_device_error_ptr();
  REORDER_REQUIRE(a.err != nullptr, "no device error word");
  auto go = [&](auto kernel, int threads_of, size_t smem) -> int {
    DSP_CUDA(launch_pdl(kernel, dim3((unsigned)blocks), dim3(threads_of), smem, stream, a));
    return 0;
  };
  if (bulk) {
    static bool allowed[MAX_DEVICES] = {};  // asked for once a device
    const int device = current_device();
    if (device < 0 || !allowed[device]) {
      DSP_CUDA(cudaFuncSetAttribute(reorder_bulk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BULK_BYTES));
      if (device >= 0) allowed[device] = true;
    }
    const int rc = go(reorder_bulk_kernel, BULK_THREADS, (size_t)(n * chunk_bytes));
    if (rc != 0) return rc;
  } else {
    const int rc = threads == 256 ? (piece == 16 ? go(reorder_kernel<uint4, 256>, 256, 0) : piece == 4 ? go(reorder_kernel<uint32_t, 256>, 256, 0)
                                                                                                       : go(reorder_kernel<uint16_t, 256>, 256, 0))
                                  : (piece == 16 ? go(reorder_kernel<uint4, 1024>, 1024, 0) : piece == 4 ? go(reorder_kernel<uint32_t, 1024>, 1024, 0)
                                                                                                         : go(reorder_kernel<uint16_t, 1024>, 1024, 0));
    if (rc != 0) return rc;
  }
  DSP_CHECK_LAUNCH("reorder_slots");
  return 0;
}
