// Attention of drafted trees over the paged key/value cache, 32-bit arithmetic, and the merge of partial results.
//
// Node i of tree s has its key and value at place ctx_s + i of the request's cache.  It sees the stored keys
// j < ctx_s and, of the tree, the nodes k whose bit is set in visible[row of i] (its ancestors and itself):
//     o_i = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q_i . k_j)
// With window W, node i at depth d_i sits at position ctx_s + d_i and sees positions above ctx_s + d_i - W only.  A row
// that sees nothing gives 0.  The work is cut as tree_schedule.cuh says.
#include "merge_parts.cuh"
#include "rows_attn.cuh"
#include "tensor_checks.cuh"
#include "tree_schedule.cuh"

namespace {
using namespace tree;

// Every block makes out which CTAs began an item that others share (one read of the list, a thread each), and the threads of the
// whole grid take those items' rows in turn, four columns each.  A row's partial results are asked for eight at a time, maxima,
// sums and outputs together: two latencies stand between the wait and the store.  (3 to 6 us of a call.  Merging in the main
// kernel, by the CTA that leaves an item's last part, was slower: one tree 18.8 us for 11.5.)
constexpr int COMBINE_THREADS = 256, COMBINE_WARPS = COMBINE_THREADS / 32, COMBINE_BLOCKS_PER_SM = 4;
template <typename T>
__global__ void __launch_bounds__(COMBINE_THREADS, COMBINE_BLOCKS_PER_SM)
tree_combine_kernel(const TreeScratch scratch, T* __restrict__ out, long out_stride, int G, int D, int R, int ctas) {
  __shared__ int items[COMBINE_THREADS];  // CTAs that began one
  __shared__ int of_warp[COMBINE_WARPS], rows_of_warp[COMBINE_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  for (int c0 = 0; c0 < ctas; c0 += COMBINE_THREADS) {
    const bool has = c0 + tid < ctas && scratch.splits[c0 + tid].parts > 0;
    const int most_rows = __reduce_max_sync(0xffffffffu, has ? scratch.splits[c0 + tid].rows : 0);
    // the same list in every block: in the order of the CTAs
    const uint32_t those = __ballot_sync(0xffffffffu, has);
    __syncthreads();
    if (lane == 0) {
      of_warp[warp] = __popc(those);
      rows_of_warp[warp] = most_rows;
    }
    __syncthreads();
    int before = 0, n_items = 0, rows = 0;
#pragma unroll
    for (int w = 0; w < COMBINE_WARPS; ++w) {
      before += w < warp ? of_warp[w] : 0;
      n_items += of_warp[w];
      rows = max(rows, rows_of_warp[w]);
    }
    if (has) items[before + __popc(those & ((1u << lane) - 1u))] = c0 + tid;
    __syncthreads();
    const int quads = D / 4, pieces = n_items * rows * quads;
    for (int i = blockIdx.x * COMBINE_THREADS + tid; i < pieces; i += gridDim.x * COMBINE_THREADS) {
      // neighbouring threads take neighbouring columns and rows
      const int row = i / quads, d = (i - row * quads) * 4, c = items[row / rows], r = row % rows;
      const Split x = scratch.splits[c];
      if (r >= x.rows) continue;
      const float2* ml = reinterpret_cast<const float2*>(scratch.part_ml);
      auto row_of = [&](int k) -> size_t { return (k == 0 ? 2 * (size_t)c + 1 : 2 * (size_t)(c + k)) * R + r; };  // of the k-th part
      const int rr = x.row0 + r;
      T* dst = out + (size_t)(x.first + rr / G) * out_stride + (size_t)(x.head * G + rr % G) * D;
      store4(dst + d, merged(merge_parts(x.parts, [&](int k, float2& m, float4& v) {
        const size_t at = row_of(k);
        m = ml[at];
        v = load4(scratch.part_o + at * D + d);
      })));
    }
  }
}
}  // namespace

cudaError_t tree_combine(const TreeScratch& scratch, void* out, long out_stride, int G, int D, int rows_per_tile, int ctas,
                         int dtype, cudaStream_t stream) {
  const int sms = dsp_num_sms();
  const dim3 grid((unsigned)min((long)ctas * rows_per_tile / COMBINE_WARPS, (long)(sms > 0 ? sms : 1) * COMBINE_BLOCKS_PER_SM));
  return dtype == DSP_F32 ? launch_pdl(tree_combine_kernel<float>, grid, dim3(COMBINE_THREADS), 0, stream, scratch, (float*)out,
                                       out_stride, G, D, rows_per_tile, ctas)
                          : launch_pdl(tree_combine_kernel<bf16>, grid, dim3(COMBINE_THREADS), 0, stream, scratch, (bf16*)out,
                                       out_stride, G, D, rows_per_tile, ctas);
}

struct DspTreeOptions {  // as ops/tree.py packs them
  long max_nodes, window, sms, tensor_cores;
  double scale;
};

// tensors: q, key pool, value pool, page table, ctx_len, node_start, depth (or none), visible, out, scratch.  `tensor_cores`:
// address of the tensor-core kernel's entry point for this head size, or 0.
extern "C" int dsp_tree_attention(const DspTensor* t, const DspTreeOptions* o, cudaStream_t stream) {
  const DspTensor &q = t[0], &k = t[1], &v = t[2], &table = t[3], &ctx = t[4], &start = t[5], &depth = t[6], &visible = t[7],
                  &out = t[8], &scratch = t[9];
  DSP_REQUIRE(q.device >= 0, "tree_attention: CUDA tensors only (there is no CPU path)");
  DSP_REQUIRE(q.dims == 2 && k.dims == 4 && v.dims == 4, "tree_attention: q [T, H * D] and two pools [pages, heads, page_size, D] expected");
  const long T = q.size[0], columns = q.size[1], pages = k.size[0], KVH = k.size[1], page = k.size[2], D = k.size[3];
  DSP_REQUIRE(q.dtype == DSP_T_F32 || q.dtype == DSP_T_BF16, "tree_attention: kernels exist for float32 and bfloat16");
  DSP_REQUIRE(k.dtype == q.dtype && v.dtype == q.dtype && k.device == q.device && v.device == q.device && k.contiguous && v.contiguous &&
                  v.size[0] == pages && v.size[1] == KVH && v.size[2] == page && v.size[3] == D,
              "tree_attention: the pools must be contiguous, alike, and of the type and on the device of q");
  DSP_REQUIRE(T == 0 || q.stride[1] == 1 || columns == 1, "tree_attention: the columns of q must be neighbours");
  DSP_REQUIRE(D % 8 == 0 && D >= 8 && D <= 256 && KVH > 0 && columns > 0 && columns % D == 0 && columns / D % KVH == 0,
              "tree_attention: %ld query columns on %ld heads of %ld (a multiple of 8 up to 256)", columns, KVH, D);
  DSP_REQUIRE(ctx.dims == 1, "tree_attention: ctx_len must be one-dimensional");
  const long S = ctx.size[0], words = visible.dims == 2 ? visible.size[1] : 0;
  DSP_REQUIRE(tensor_is(visible, DSP_T_I64, q.device, 2, T, words) && words >= 1 && 64 * words >= o->max_nodes,
              "tree_attention: visible must be contiguous int64 [%ld, words] with a bit for each of %ld nodes", T, o->max_nodes);
  DSP_REQUIRE(is_scale(o->scale) && o->window >= 0 && o->window <= 0x7fffffff && o->max_nodes >= 1,
              "tree_attention: scale %g must be positive and finite in 32 bits, window %ld not negative, max_nodes %ld at least 1", o->scale, o->window,
              o->max_nodes);
  DSP_REQUIRE(tensor_is(ctx, DSP_T_I32, q.device, 1, S) && tensor_is(start, DSP_T_I32, q.device, 1, S + 1),
              "tree_attention: ctx_len [%ld] and node_start [%ld] must be contiguous int32 on the device of q", S, S + 1);
  DSP_REQUIRE(is_page_table(table, q.device, S), "tree_attention: page_table must be int32 [%ld, pages], neighbouring pages side by side", S);
  DSP_REQUIRE(depth.dims < 0 ? o->window == 0 : tensor_is(depth, DSP_T_I32, q.device, 1, T),
              "tree_attention: depth must be contiguous int32 [%ld]; a window needs it", T);
  DSP_REQUIRE(out.dtype == q.dtype && out.device == q.device && out.dims == 2 && out.size[0] == T && out.size[1] == columns &&
                  (T == 0 || out.stride[1] == 1 || columns == 1),
              "tree_attention: out must be like the queries [%ld, %ld] with neighbouring columns", T, columns);
  DSP_REQUIRE(T <= 0x7fffffff && S <= 0x7fffffff && pages <= 0x7fffffff && page >= 1 && o->sms >= 1, "tree_attention: sizes out of range");
  if (T == 0 || S == 0) return 0;
  const uintptr_t bits = (uintptr_t)q.data | (uintptr_t)k.data | (uintptr_t)v.data | (uintptr_t)out.data;
  const long piece = q.dtype == DSP_T_F32 ? 4 : 8;  // elements of 16 bytes
  DSP_REQUIRE(bits % 16 == 0 && (T == 1 || (q.stride[0] % piece == 0 && out.stride[0] % piece == 0)),
              "tree_attention: rows must begin on 16 bytes");
  // the tensor-core kernel is built for these page sizes; everything else takes the 32-bit kernel
  const bool tensor_cores = o->tensor_cores != 0 && q.dtype == DSP_T_BF16 && (D == 64 || D == 128) &&
                            (page == 8 || page == 16 || page == 32 || page == 64) && pages > 0;
  const long G = columns / D / KVH, rows = tensor_cores ? 1 << ROW_SHIFT_TENSOR_CORES : ROWS;
  // a multiple of the row tiles that trees have: then those of one head read its keys at the same time
  const long row_tiles = (o->max_nodes * G + rows - 1) / rows;
  const long places = o->sms * (tensor_cores || D > 128 ? 1 : 2);  // (by shared memory two CTAs of the 32-bit kernel an SM)
  const long ctas = row_tiles < places ? places - places % row_tiles : places;
  // Key tiles are counted in 32 bits: those of all trees, each with as many stored tokens as its pages hold.
  const long most_ctx = min(table.size[1] * page, 1L << 30);
  DSP_REQUIRE(T * G <= 0x7fffffff && (T * G / rows + S) * KVH <= 0x7fffffff / ((most_ctx + T) / KEYS_PER_TILE + 1),
              "tree_attention: %ld rows of %ld heads over pages for %ld tokens a request are too many for one call", T, G, most_ctx);
  DSP_REQUIRE(scratch.contiguous && scratch.device == q.device && scratch.dims == 1 && (uintptr_t)scratch.data % 16 == 0 &&
                  scratch.size[0] >= 2 * ctas * rows * (D + 2) + 8 * ctas,
              "tree_attention: scratch is too small");
  DspTreeAttention a = {};
  a.sh.node_start = (const int*)start.data;
  a.sh.ctx_len = (const int*)ctx.data;
  a.sh.S = (int)S;
  a.sh.KVH = (int)KVH;
  a.sh.G = (int)G;
  a.sh.row_shift = tensor_cores ? ROW_SHIFT_TENSOR_CORES : ROW_SHIFT;
  a.sh.window = (int)o->window;
  a.sh.rows = (int)T;
  a.sh.most_ctx = (int)most_ctx;
  a.q = q.data;
  a.k_pool = k.data;
  a.v_pool = v.data;
  a.page_table = (const int*)table.data;
  a.depth = depth.dims < 0 ? nullptr : (const int*)depth.data;
  a.visible = (const unsigned long long*)visible.data;
  a.out = out.data;
  a.scratch = tree_scratch((float*)scratch.data, ctas, rows, D);
  a.q_stride = q.stride[0];
  a.out_stride = out.stride[0];
  a.pt_stride = (int)table.stride[0];
  a.table_width = (int)table.size[1];
  a.words = (int)words;
  a.D = (int)D;
  a.page_size = (int)page;
  a.num_pages = (int)pages;
  a.ctas = (int)ctas;
  a.scale = (float)o->scale;
  a.err = a.sh.err = dsp_device_error_ptr();
  DSP_REQUIRE(a.err != nullptr, "tree_attention: no device error word");
  if (tensor_cores) {
    typedef int (*Kernel)(const DspTreeAttention*, cudaStream_t);
    const int rc = reinterpret_cast<Kernel>(o->tensor_cores)(&a, stream);
    DSP_REQUIRE(rc == 0, "tree_attention: %s", rc == 4 ? "shared memory opt-in or tensor map creation failed" : "launch failed");
  } else {
    a.sh.min_units = 1;
    const int rc = q.dtype == DSP_T_F32 ? launch_rows_attn<TreeWork, float>(a, stream) : launch_rows_attn<TreeWork, bf16>(a, stream);
    if (rc != 0) return rc;
  }
  DSP_CUDA(tree_combine(a.scratch, a.out, a.out_stride, a.sh.G, a.D, (int)rows, a.ctas, q.dtype == DSP_T_F32 ? DSP_F32 : DSP_BF16, stream));
  DSP_CHECK_LAUNCH("tree_attention");
  return 0;
}
