// The accepted branch of a drafted tree is put into line in the paged cache: the keys and values (whatever a layer keeps
// per token) of node path[j] move from place ctx + path[j] to ctx + j, in every layer cache and pool.
//
// A path ascends, so path[j] >= j and a place is written only after what lay there has been read, if a thread moves its
// piece of the nodes in order.  The rows are copied as they are; nothing is computed.
#include "common.cuh"

namespace {
constexpr int MAX_POOLS = 8;

struct Pool {
  unsigned char* data;  // [layers][pages][heads][page_size][row_bytes]
  int layers, heads, pieces;  // pieces of 16 bytes a row
  long layer_bytes;
  int num_pages;
};
struct Args {
  Pool pool[MAX_POOLS];
  const int *page_table, *ctx_len, *path, *count;
  int pt_stride, path_stride, path_width, page_size, pools;
  int* err;
};

// block: (layer of all pools, tree)
__global__ void __launch_bounds__(256)
tree_keep_kernel(const Args a) {
  const int s = blockIdx.y;
  const int* path = a.path + (size_t)s * a.path_stride;
  const int n = min(a.count[s], a.path_width), ctx = a.ctx_len[s];
  const int* table = a.page_table + (size_t)s * a.pt_stride;
  int layer = blockIdx.x, which = 0;
  while (layer >= a.pool[which].layers) layer -= a.pool[which++].layers;
  const Pool p = a.pool[which];
  unsigned char* base = p.data + (size_t)layer * p.layer_bytes;
  const size_t row = (size_t)p.pieces * 16;
  auto place = [&](int key, int head) -> long {
    if (key < 0 || key / a.page_size >= a.pt_stride) return -1;
    const int page = table[key / a.page_size];
    if (page < 0 || page >= p.num_pages) return -1;
    return (long)((((size_t)page * p.heads + head) * a.page_size + key % a.page_size) * row);
  };
  int before = -1;
  for (int j = 0; j < n; ++j) {
    const int node = path[j];
    if (node <= before) {  // not a path: nothing behind it is moved
      if (threadIdx.x == 0) atomicOr(a.err, DSP_ERR_BAD_TREE);
      return;
    }
    before = node;
    if (node == j) continue;
    for (int i = threadIdx.x; i < p.heads * p.pieces; i += blockDim.x) {
      const int head = i / p.pieces, c = i % p.pieces;
      const long from = place(ctx + node, head), to = place(ctx + j, head);
      if (from < 0 || to < 0) {
        atomicOr(a.err, DSP_ERR_BAD_PAGE);
        continue;
      }
      *reinterpret_cast<uint4*>(base + to + c * 16) = *reinterpret_cast<const uint4*>(base + from + c * 16);
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
    a.pool[i] = Pool{(unsigned char*)d[0], (int)d[1], (int)d[3], (int)(d[4] / 16), d[2] * d[3] * p->page_size * d[4], (int)d[2]};
    blocks += d[1];
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
  a.pools = (int)p->pools;
  a.err = dsp_device_error_ptr();
  DSP_REQUIRE(a.err != nullptr, "dsp_tree_keep: no device error word");
  DSP_CUDA(launch_plain(tree_keep_kernel, dim3((unsigned)blocks, (unsigned)p->S), dim3(256), 0, stream, a));
  DSP_CHECK_LAUNCH("dsp_tree_keep");
  return 0;
}
