// The accepted branch of a drafted tree is put into line in the paged cache: the keys and values (whatever a layer keeps
// per token) of node path[j] move from place ctx + path[j] to ctx + j, in every layer cache and pool.
//
// A path ascends, so path[j] >= j and a place is written only after what lay there has been read, if a thread moves its
// piece of the nodes in order, a few at a time.  The rows are copied as they are; nothing is computed.
//
// What bounds it: the bytes for large batches; for small ones the chain count, path -> page table -> row.  A block works
// that chain out once for several layers, and a thread's loads of up to eight nodes are under way together.  8 trees of 28
// layers 2.8 us; 64 trees of 48 layers with rows of 256 bytes 23.8 us, 3.8 TB/s, 0.58 of what a plain copy reaches.
#include <limits.h>

#include "tensor_checks.cuh"

namespace {
constexpr int MAX_POOLS = 8, THREADS = 128, AHEAD = 8;
// Pieces of 16 bytes that a thread moves of every node, about: a block takes layers enough for that.  Few, where the SMs have room
// for all blocks then (six an SM), since a thread takes them one after the other (8 trees of 28 layers: 2.8 us with one, 3.5 with
// two, 5.4 with four); four otherwise, for the chain's sake (64 trees of 48 layers: 27.5, 24.3, 23.8).
constexpr int FEW = 1, MANY = 4, BLOCKS_PER_SM = 6;

struct Pool {
  unsigned char* data;  // [layers][pages][heads][page_size][row_bytes]
  int layers, heads, pieces;  // pieces of 16 bytes a row
  int layers_per_block, blocks;
  long layer_bytes;
  int num_pages;
};
struct Args {
  Pool pool[MAX_POOLS];
  const int *page_table, *ctx_len, *path, *count;
  int pt_stride, table_width, path_stride, path_width, page_size;
  int* err;
};

// block: (group of layers of one pool, tree)
__global__ void __launch_bounds__(THREADS)
tree_keep_kernel(const __grid_constant__ Args a) {
  __shared__ int from_page[THREADS], from_at[THREADS], to_page[THREADS], to_at[THREADS];  // of a node; from_page -1: it stays
  __shared__ int stop;  // first node that does not come after the one in front of it
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.y, tid = threadIdx.x;
  int block = blockIdx.x, which = 0;
  while (block >= a.pool[which].blocks) block -= a.pool[which++].blocks;
  const Pool& p = a.pool[which];
  const int layer0 = block * p.layers_per_block, layers = min(p.layers_per_block, p.layers - layer0);
  const int* path = a.path + (size_t)s * a.path_stride;
  const int* table = a.page_table + (size_t)s * a.pt_stride;
  const int n = min(a.count[s], a.path_width), ctx = a.ctx_len[s];
  const int row_pieces = p.heads * p.pieces, items = layers * row_pieces;
  if (tid == 0) stop = n;
  for (int j0 = 0; j0 < n; j0 += THREADS) {
    const int j = j0 + tid;
    int from = -1;
    __syncthreads();  // (nobody reads the last nodes' places any more)
    if (j < n) {
      const int node = path[j];
      if (node <= (j > 0 ? path[j - 1] : -1)) {
        atomicMin(&stop, j);
        atomicOr(a.err, DSP_ERR_BAD_TREE);
      } else if (node != j) {
        const bool counted = ctx >= 0 && node <= INT_MAX - ctx;  // (no path has a negative node: it ascends from -1)
        const int k = counted ? ctx + node : 0, k2 = counted ? ctx + j : 0;
        const bool inside = counted && k / a.page_size < a.table_width;
        from = inside ? table[k / a.page_size] : -1;
        const int to = inside ? table[k2 / a.page_size] : -1;
        if (from < 0 || from >= p.num_pages || to < 0 || to >= p.num_pages) {
          atomicOr(a.err, DSP_ERR_BAD_PAGE);
          from = -1;
        }
        from_at[tid] = k % a.page_size;
        to_page[tid] = to;
        to_at[tid] = k2 % a.page_size;
      }
    }
    from_page[tid] = from;
    __syncthreads();
    const int nodes = min(stop, n) - j0;
    if (nodes <= 0) break;
    for (int i = tid; i < items; i += THREADS) {
      const int layer = i / row_pieces, piece = i - layer * row_pieces, head = piece / p.pieces;
      unsigned char* base = p.data + (size_t)(layer0 + layer) * p.layer_bytes + (size_t)(piece - head * p.pieces) * 16;
      const size_t row = (size_t)p.pieces * 16;
      auto at = [&](int page, int off) { return base + (((size_t)page * p.heads + head) * a.page_size + off) * row; };
      for (int c0 = 0; c0 < min(nodes, THREADS); c0 += AHEAD) {
        uint4 v[AHEAD];
#pragma unroll
        for (int c = 0; c < AHEAD; ++c)
          if (c0 + c < min(nodes, THREADS) && from_page[c0 + c] >= 0)
            v[c] = *reinterpret_cast<const uint4*>(at(from_page[c0 + c], from_at[c0 + c]));
#pragma unroll
        for (int c = 0; c < AHEAD; ++c)
          if (c0 + c < min(nodes, THREADS) && from_page[c0 + c] >= 0)
            *reinterpret_cast<uint4*>(at(to_page[c0 + c], to_at[c0 + c])) = v[c];
      }
    }
  }
}
}  // namespace

// tensors: page table, ctx_len, path, count, and so many pools [layers, pages, heads, page_size, width].
extern "C" int dsp_tree_keep(const DspTensor* t, int pools, cudaStream_t stream) {
  const DspTensor &table = t[0], &ctx = t[1], &path = t[2], &count = t[3], *pool = t + 4;
  DSP_REQUIRE(pools >= 1 && pools <= MAX_POOLS, "keep_path: %d pools (1 to %d)", pools, MAX_POOLS);
  DSP_REQUIRE(ctx.dims == 1 && path.dims == 2, "keep_path: ctx_len [S] and path [S, n] expected");
  const long S = ctx.size[0], width = path.size[1], page = pool[0].dims == 5 ? pool[0].size[3] : 0;
  const int dev = pool[0].device;
  DSP_REQUIRE(dev >= 0, "keep_path: CUDA tensors only (there is no CPU path)");
  DSP_REQUIRE(tensor_is(ctx, DSP_T_I32, dev, 1, S) && tensor_is(count, DSP_T_I32, dev, 1, S) && tensor_is(path, DSP_T_I32, dev, 2, S, width),
              "keep_path: ctx_len [%ld], count [%ld] and path [%ld, n] must be contiguous int32 on the device of the pools", S, S, S);
  DSP_REQUIRE(is_page_table(table, dev, S), "keep_path: page_table must be int32 [%ld, pages], neighbouring pages side by side", S);
  DSP_REQUIRE(S <= 65535 && width <= 0x7fffffff, "keep_path: %ld trees (at most 65,535)", S);
  Args a = {};
  long blocks = 0;
  int used = 0;
  for (int i = 0; i < pools; ++i) {
    const DspTensor& p = pool[i];
    DSP_REQUIRE(p.dims == 5 && p.contiguous && p.device == dev && p.size[3] == page && page >= 1,
                "keep_path: a pool must be contiguous [layers, pages, heads, %ld, width] on the device of the others", page);
    DSP_REQUIRE(p.dtype == DSP_T_F32 || p.dtype == DSP_T_BF16, "keep_path: pools are float32 or bfloat16");
    const long layers = p.size[0], pages = p.size[1], heads = p.size[2], row = p.size[4] * (p.dtype == DSP_T_F32 ? 4 : 2);
    DSP_REQUIRE(row % 16 == 0 && row > 0 && (uintptr_t)p.data % 16 == 0, "keep_path: rows of %ld bytes (whole 16-byte pieces are moved)", row);
    if (layers == 0 || heads == 0) continue;  // (a pool without rows has no blocks)
    a.pool[used++] = Pool{(unsigned char*)p.data, (int)layers, (int)heads, (int)(row / 16), 0, 0, pages * heads * page * row, (int)pages};
  }
  const long places = (long)dsp_num_sms() * BLOCKS_PER_SM;
  for (int items = FEW; items <= MANY; items *= 2) {
    blocks = 0;
    for (int i = 0; i < used; ++i) {
      Pool& p = a.pool[i];
      p.layers_per_block = (int)min((long)p.layers, max(1L, (long)items * THREADS / ((long)p.heads * p.pieces)));
      p.blocks = (p.layers + p.layers_per_block - 1) / p.layers_per_block;
      blocks += p.blocks;
    }
    if (blocks * S <= places) break;
  }
  if (S == 0 || width == 0 || blocks == 0) return 0;
  a.page_table = (const int*)table.data;
  a.ctx_len = (const int*)ctx.data;
  a.path = (const int*)path.data;
  a.count = (const int*)count.data;
  a.pt_stride = (int)table.stride[0];
  a.table_width = (int)table.size[1];
  a.path_stride = (int)path.stride[0];
  a.path_width = (int)width;
  a.page_size = (int)page;
  a.err = dsp_device_error_ptr();
  DSP_REQUIRE(a.err != nullptr, "keep_path: no device error word");
  DSP_CUDA(launch_pdl(tree_keep_kernel, dim3((unsigned)blocks, (unsigned)S), dim3(THREADS), 0, stream, a));
  DSP_CHECK_LAUNCH("keep_path");
  return 0;
}
