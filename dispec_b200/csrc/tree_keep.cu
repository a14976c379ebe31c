// The accepted branch of a drafted tree is put into line in the paged cache: the keys and values (whatever a layer keeps
// per token) of node path[j] move from place ctx + path[j] to ctx + j, in every layer cache and pool.
//
// A path ascends, so path[j] >= j and a place is written only after what lay there has been read, if a thread moves its
// piece of the nodes in order, a few at a time.  The rows are copied as they are; nothing is computed.
//
// What bounds it: the bytes for large batches; for small ones the chain count, path -> page table -> row.  A block works
// that chain out once for several layers, and a thread's loads of up to eight nodes are under way together.
#include "common.cuh"

namespace {
constexpr int MAX_POOLS = 8, THREADS = 256, AHEAD = 8;
constexpr int ITEMS = 2;  // pieces of 16 bytes that a thread moves of every node, about: a block takes layers enough for that

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
  int pt_stride, path_stride, path_width, page_size;
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
        const int k = ctx + node, k2 = ctx + j;
        const bool inside = ctx >= 0 && k / a.page_size < a.pt_stride;
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

// What the Python side packs, in this order (ops/tree.py); `pool` holds (address, layers, pages, heads, bytes of a row).
struct DspTreeKeep {
  const int *page_table, *ctx_len, *path, *count;
  long pt_stride, path_stride, path_width, page_size, S, pools;
  long pool[MAX_POOLS][5];
};

extern "C" int dsp_tree_keep(const DspTreeKeep* p, cudaStream_t stream) {
  if (p->S == 0 || p->pools == 0) return 0;
  DSP_REQUIRE(p->S > 0 && p->S <= 65535 && p->pools > 0 && p->pools <= MAX_POOLS && p->page_size >= 1 && p->path_width >= 1,
              "dsp_tree_keep: %ld trees, %ld pools", p->S, p->pools);
  Args a = {};
  long blocks = 0;
  for (int i = 0; i < p->pools; ++i) {
    const long* d = p->pool[i];
    DSP_REQUIRE(d[4] % 16 == 0 && d[0] % 16 == 0 && d[4] > 0, "dsp_tree_keep: rows of %ld bytes (whole 16-byte pieces)", d[4]);
    if (d[1] == 0 || d[3] == 0) continue;  // (a pool without rows has no blocks)
    const int row_pieces = (int)(d[3] * d[4] / 16), per = min((int)d[1], max(1, ITEMS * THREADS / row_pieces));
    a.pool[i] = Pool{(unsigned char*)d[0], (int)d[1], (int)d[3], (int)(d[4] / 16), per, ((int)d[1] + per - 1) / per,
                     d[2] * d[3] * p->page_size * d[4], (int)d[2]};
    blocks += a.pool[i].blocks;
  }
  if (blocks == 0) return 0;
  a.page_table = p->page_table;
  a.ctx_len = p->ctx_len;
  a.path = p->path;
  a.count = p->count;
  a.pt_stride = (int)p->pt_stride;
  a.path_stride = (int)p->path_stride;
  a.path_width = (int)p->path_width;
  a.page_size = (int)p->page_size;
  a.err = dsp_device_error_ptr();
  DSP_REQUIRE(a.err != nullptr, "dsp_tree_keep: no device error word");
  DSP_CUDA(launch_pdl(tree_keep_kernel, dim3((unsigned)blocks, (unsigned)p->S), dim3(THREADS), 0, stream, a));
  DSP_CHECK_LAUNCH("dsp_tree_keep");
  return 0;
}
