// Attention of drafted trees over the paged key/value cache, 32-bit arithmetic, and the merge of partial results.
//
// Node i of tree s has its key and value at place ctx_s + i of the request's cache.  It sees the stored keys
// j < ctx_s and, of the tree, the nodes k whose bit is set in visible[row of i] (its ancestors and itself):
//     o_i = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q_i . k_j)
// With window W, node i at depth d_i sits at position ctx_s + d_i and sees positions above ctx_s + d_i - W only.  A row
// that sees nothing gives 0.  The work is cut as tree_schedule.cuh says.
//
// A block holds 32 rows and walks key tiles of 64, queries, keys and values as floats in shared memory: thread
// (ty, tx) of 16 x 16 owns rows ty, ty + 16 and keys tx + 16 j of the scores, and of the result the same rows and
// the dimensions 4 tx .. 4 tx + 3 of each 64.  Maximum and sum of a row are exchanged between its 16 threads by
// shuffles.  Multiply-adds and the reads from shared memory that feed them (5 for every 16, two cycles each) bound it: for 8
// trees of 32 nodes behind 4,000 tokens, 12 heads of 128 on 2, 32-bit, 223 us, 21 TFLOP/s.  Up to head size 128 two blocks
// share an SM, so that one's copies and softmax run beside the other's products (513 us with one, whose rows were copied
// between barriers); keys and values come while the tile before is still being used.
#include <type_traits>

#include "tensor_checks.cuh"
#include "tree_schedule.cuh"

namespace {
using namespace tree;

constexpr int ROW_SHIFT = 5, ROWS = 1 << ROW_SHIFT, KEYS = KEYS_PER_TILE, TX = 16, THREADS = 256, RI = ROWS / 16, KJ = KEYS / TX, LP = KEYS + 4;

typedef DspTreeAttention Args;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const bf16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(bf16* p, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  uint2 u;
  u.x = *reinterpret_cast<const uint32_t*>(&a);
  u.y = *reinterpret_cast<const uint32_t*>(&b);
  *reinterpret_cast<uint2*>(p) = u;
}

// A key tile's rows on their way into shared memory: 32-bit elements by asynchronous copies, 16-bit ones through registers, asked
// for together and stored (`put`) a step later.  A row takes 16 DJ lanes, four elements each, or a warp twice.
template <typename T, int DJ>
struct Rows {
  static constexpr int LANES = DJ == 1 ? 16 : 32, AT_ONCE = THREADS / LANES, COLS = DJ * 16 / LANES, N = KEYS / AT_ONCE;
  uint2 x[sizeof(T) == 2 ? N * COLS : 1];
  int row, col;
  __device__ __forceinline__ Rows() : row(threadIdx.x / LANES), col(threadIdx.x % LANES * 4) {}
  __device__ __forceinline__ void ask(const T* pool, const long* slots, float* dst, int D, int LD) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const long at = slots[row + n * AT_ONCE];
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const int d = col + c * 128;
        if constexpr (sizeof(T) == 2) {
          x[n * COLS + c] = make_uint2(0u, 0u);
          if (at >= 0 && d < D) x[n * COLS + c] = __ldg(reinterpret_cast<const uint2*>(pool + at * D + d));
        } else if (d < D) {
          // (no bytes are read for a key that is not there: zeros)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst + (row + n * AT_ONCE) * LD + d)),
                       "l"(pool + (at < 0 ? 0 : at * D + d)), "r"(at < 0 ? 0 : 16)
                       : "memory");
        }
      }
    }
    if constexpr (sizeof(T) == 4) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void put(float* dst, int D, int LD) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const int d = col + c * 128;
          const uint2 u = x[n * COLS + c];
          const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
          const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
          if (d < D) *reinterpret_cast<float4*>(dst + (row + n * AT_ONCE) * LD + d) = make_float4(a.x, a.y, b.x, b.y);
        }
    }
  }
  // all copies but the newest `PENDING` groups are there (for this thread; a barrier makes them everybody's)
  template <int PENDING>
  static __device__ __forceinline__ void wait() {
    if constexpr (sizeof(T) == 4) asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
  }
};

// DJ: 64-wide slices of the head dimension
template <typename T, int DJ>
__global__ void __launch_bounds__(THREADS, DJ == 4 ? 1 : 2)
tree_attn_kernel(const Args a) {
  extern __shared__ float smem[];
  const int D = a.D, LD = D + 4, tid = threadIdx.x, tx = tid % TX, ty = tid / TX;
  float* qs = smem;              // [ROWS][LD]
  float* ks = qs + ROWS * LD;    // [KEYS][LD]
  float* vs = ks + KEYS * LD;    // [KEYS][LD]
  float* ps = vs + KEYS * LD;    // [ROWS][LP]
  __shared__ long slots_of_keys[2][KEYS];  // of this key tile and the coming one
  const Shape& sh = a.sh;
  Walk w;
  pdl_launch_dependents();
  pdl_wait();
  if (!w.begin(sh, blockIdx.x, gridDim.x)) {
    if (tid == 0) a.scratch.splits[w.cta].parts = 0;
    return;
  }
  const int G = sh.G;
  bool more;
  do {
    const Share& t = w.at;
    const int row0 = t.row_tile * ROWS, rows = min(ROWS, t.n * G - row0);
    const int total = t.ctx + t.n;
    const int* table = a.page_table + (size_t)t.seq * a.pt_stride;
    auto find_keys = [&](int kt) {
      const int key = kt * KEYS + tid;
      long at = -1;
      if (key < total && (sh.window <= 0 || key > t.ctx - sh.window)) {
        const int page = key / a.page_size < a.table_width ? table[key / a.page_size] : -1;
        if (page >= 0 && page < a.num_pages)
          at = ((long)page * sh.KVH + t.head) * a.page_size + key % a.page_size;
        else
          atomicOr(a.err, DSP_ERR_BAD_PAGE);
      }
      slots_of_keys[kt & 1][tid] = at;
    };
    __syncthreads();
    if (tid < KEYS) find_keys(t.kt_begin);
    __syncthreads();
    Rows<T, DJ> k_rows, v_rows;
    k_rows.ask((const T*)a.k_pool, slots_of_keys[t.kt_begin & 1], ks, D, LD);
    v_rows.ask((const T*)a.v_pool, slots_of_keys[t.kt_begin & 1], vs, D, LD);
    {
      constexpr int LANES = Rows<T, DJ>::LANES, AT_ONCE = Rows<T, DJ>::AT_ONCE;
#pragma unroll
      for (int r0 = 0; r0 < ROWS; r0 += AT_ONCE)
#pragma unroll
        for (int c = 0; c < Rows<T, DJ>::COLS; ++c) {
          const int r = r0 + tid / LANES, d = tid % LANES * 4 + c * 128, rr = row0 + r;
          if (d >= D) continue;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < rows) v = load4((const T*)a.q + (size_t)(t.first + rr / G) * a.q_stride + (size_t)(t.head * G + rr % G) * D + d);
          *reinterpret_cast<float4*>(qs + r * LD + d) = v;
        }
    }
    float m[RI], l[RI], acc[RI][4 * DJ];
    int depth[RI], node[RI];
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = ty + i * 16;
      node[i] = r < rows ? t.first + (row0 + r) / G : -1;
      depth[i] = (sh.window > 0 && node[i] >= 0) ? a.depth[node[i]] : 0;
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < 4 * DJ; ++d) acc[i][d] = 0.f;
    }
    k_rows.put(ks, D, LD);
    // the coming tile's keys are asked for when this one's have been used, before the softmax, and its values at the end
    for (int kt = t.kt_begin; kt < t.kt_end; ++kt) {
      const int key0 = kt * KEYS;
      const bool another = kt + 1 < t.kt_end;
      const long* slot_of_key = slots_of_keys[kt & 1];
      Rows<T, DJ>::template wait<1>();
      __syncthreads();
      if (tid < KEYS && another) find_keys(kt + 1);  // (its page id arrives during the products)
      float s[RI][KJ];
#pragma unroll
      for (int i = 0; i < RI; ++i)
#pragma unroll
        for (int j = 0; j < KJ; ++j) s[i][j] = 0.f;
      for (int d = 0; d < D; d += 4) {
        float4 x[RI];
#pragma unroll
        for (int i = 0; i < RI; ++i) x[i] = *reinterpret_cast<const float4*>(qs + (ty + i * 16) * LD + d);
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const float4 y = *reinterpret_cast<const float4*>(ks + (tx + j * TX) * LD + d);
#pragma unroll
          for (int i = 0; i < RI; ++i)
            s[i][j] = fmaf(x[i].x, y.x, fmaf(x[i].y, y.y, fmaf(x[i].z, y.z, fmaf(x[i].w, y.w, s[i][j]))));
        }
      }
      v_rows.put(vs, D, LD);
      Rows<T, DJ>::template wait<0>();
      __syncthreads();
      if (another) k_rows.ask((const T*)a.k_pool, slots_of_keys[(kt + 1) & 1], ks, D, LD);
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const int key = key0 + tx + j * TX;
          bool seen = node[i] >= 0 && slot_of_key[tx + j * TX] >= 0;
          int depth_of_key = key - t.ctx;
          if (seen && key >= t.ctx) {
            const int k = key - t.ctx;
            seen = k < 64 * a.words && ((a.visible[(size_t)node[i] * a.words + (k >> 6)] >> (k & 63)) & 1ull);
            if (sh.window > 0) depth_of_key = a.depth[t.first + k];
          }
          if (sh.window > 0) seen = seen && depth_of_key > depth[i] - sh.window;
          s[i][j] = seen ? s[i][j] * a.scale : -INFINITY;
          top = fmaxf(top, s[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m[i], top);
        const float alpha = m_new == -INFINITY ? 1.f : expf(m[i] - m_new);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const float e = s[i][j] == -INFINITY ? 0.f : expf(s[i][j] - m_new);
          ps[(ty + i * 16) * LP + tx + j * TX] = e;
          sum += e;
        }
        l[i] = l[i] * alpha + sum;  // of this thread's keys
        m[i] = m_new;
#pragma unroll
        for (int d = 0; d < 4 * DJ; ++d) acc[i][d] *= alpha;
      }
      __syncwarp();  // a row's weights are written and read by the same half warp
      auto add_values = [&](auto all_seen) {
#pragma unroll 2
        for (int j0 = 0; j0 < KEYS; j0 += 4) {
          float e[RI][4];
#pragma unroll
          for (int i = 0; i < RI; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(ps + (ty + i * 16) * LP + j0);
            e[i][0] = x.x, e[i][1] = x.y, e[i][2] = x.z, e[i][3] = x.w;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < DJ; ++c) {
              const float4 v = *reinterpret_cast<const float4*>(vs + (j0 + j) * LD + min(c * 64 + tx * 4, D - 4));
#pragma unroll
              for (int i = 0; i < RI; ++i) {
                // a hidden key's value, whatever it is, is not part of the sum
                if (!all_seen() && e[i][j] == 0.f) continue;
                acc[i][4 * c] = fmaf(e[i][j], v.x, acc[i][4 * c]);
                acc[i][4 * c + 1] = fmaf(e[i][j], v.y, acc[i][4 * c + 1]);
                acc[i][4 * c + 2] = fmaf(e[i][j], v.z, acc[i][4 * c + 2]);
                acc[i][4 * c + 3] = fmaf(e[i][j], v.w, acc[i][4 * c + 3]);
              }
            }
        }
      };
      // (no node is deeper than the tree has nodes; a page that is not there has values of zero)
      if (key0 + KEYS <= t.ctx && (sh.window <= 0 || key0 > t.ctx + t.n - 1 - sh.window))
        add_values(std::true_type());
      else
        add_values(std::false_type());
      if (another) {
        k_rows.put(ks, D, LD);
        __syncthreads();
        v_rows.ask((const T*)a.v_pool, slots_of_keys[(kt + 1) & 1], vs, D, LD);
      }
    }
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = ty + i * 16;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
      if (r >= rows) continue;
      const int rr = row0 + r;
      const float inv = t.slot >= 0 ? 1.f : l[i] > 0.f ? 1.f / l[i] : 0.f;
#pragma unroll
      for (int c = 0; c < DJ; ++c) {
        const int d = c * 64 + tx * 4;
        if (d >= D) continue;
        const float4 v = make_float4(acc[i][4 * c] * inv, acc[i][4 * c + 1] * inv, acc[i][4 * c + 2] * inv,
                                     acc[i][4 * c + 3] * inv);
        if (t.slot >= 0)
          store4(a.scratch.part_o + ((size_t)t.slot * ROWS + r) * D + d, v);
        else
          store4((T*)a.out + (size_t)(t.first + rr / G) * a.out_stride + (size_t)(t.head * G + rr % G) * D + d, v);
      }
      if (t.slot >= 0 && tx == 0)
        reinterpret_cast<float2*>(a.scratch.part_ml)[(size_t)t.slot * ROWS + r] = make_float2(m[i] * 1.4426950408889634f, l[i]);
    }
    const Split split = w.split(sh);
    more = w.next(sh);
    if (!more && tid == 0) a.scratch.splits[w.cta] = split;
  } while (more);
}

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
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k0 = 0; k0 < x.parts; k0 += 8) {
        float4 v[8];
        float2 p[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const size_t at = row_of(min(k0 + k, x.parts - 1));
          p[k] = ml[at];
          v[k] = load4(scratch.part_o + at * D + d);
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k0 + k >= x.parts) p[k] = make_float2(-INFINITY, 0.f);
          top = fmaxf(top, p[k].x);
          // a part without a largest score saw no key, and its sum is 0; or scores that are no numbers, and neither is its sum
          if (p[k].x == -INFINITY) L += p[k].y;
        }
        if (top == -INFINITY) continue;
        const float w0 = exp2f(M - top);
        L *= w0;
        acc = make_float4(acc.x * w0, acc.y * w0, acc.z * w0, acc.w * w0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (p[k].x == -INFINITY) continue;
          const float w = exp2f(p[k].x - top);
          L = fmaf(w, p[k].y, L);
          acc = make_float4(fmaf(w, v[k].x, acc.x), fmaf(w, v[k].y, acc.y), fmaf(w, v[k].z, acc.z), fmaf(w, v[k].w, acc.w));
        }
        M = top;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;  // (NaN stays)
      store4(dst + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
  }
}

template <typename T>
int launch(const Args& a, cudaStream_t stream) {
  const size_t smem = (size_t)((ROWS + 2 * KEYS) * (a.D + 4) + ROWS * LP) * sizeof(float);
  auto go = [&](auto kernel) -> int {
    DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    DSP_CUDA(launch_pdl(kernel, dim3((unsigned)a.ctas), dim3(THREADS), smem, stream, a));
    return 0;
  };
  return a.D <= 64 ? go(tree_attn_kernel<T, 1>) : a.D <= 128 ? go(tree_attn_kernel<T, 2>) : go(tree_attn_kernel<T, 4>);
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
  DSP_REQUIRE(o->scale > 0. && o->window >= 0 && o->window <= 0x7fffffff && o->max_nodes >= 1,
              "tree_attention: scale %g must be positive, window %ld not negative, max_nodes %ld at least 1", o->scale, o->window,
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
    const int rc = q.dtype == DSP_T_F32 ? launch<float>(a, stream) : launch<bf16>(a, stream);
    if (rc != 0) return rc;
  }
  DSP_CUDA(tree_combine(a.scratch, a.out, a.out_stride, a.sh.G, a.D, (int)rows, a.ctas, q.dtype == DSP_T_F32 ? DSP_F32 : DSP_BF16, stream));
  DSP_CHECK_LAUNCH("tree_attention");
  return 0;
}
