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
// shuffles.
#include "tree_schedule.cuh"

namespace {
using namespace tree;

constexpr int ROWS = 32, KEYS = 64, TX = 16, THREADS = 256, RI = ROWS / 16, KJ = KEYS / TX, LP = KEYS + 4;

struct Args {
  Shape sh;
  const void *q, *k_pool, *v_pool;
  const int *page_table, *depth;
  const unsigned long long* visible;
  void* out;
  TreeScratch scratch;
  long q_stride, out_stride;
  int pt_stride, words, D, page_size, num_pages;
  float scale;
  int* err;
};

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

// DJ: 64-wide slices of the head dimension
template <typename T, int DJ>
__global__ void __launch_bounds__(THREADS)
tree_attn_kernel(const Args a) {
  extern __shared__ float smem[];
  const int D = a.D, LD = D + 4, tid = threadIdx.x, tx = tid % TX, ty = tid / TX, cta = blockIdx.x;
  float* qs = smem;              // [ROWS][LD]
  float* ks = qs + ROWS * LD;    // [KEYS][LD]
  float* vs = ks + KEYS * LD;    // [KEYS][LD]
  float* ps = vs + KEYS * LD;    // [ROWS][LP]
  __shared__ long slot_of_key[KEYS];
  const Shape& sh = a.sh;
  Walk w;
  if (!w.begin(sh, cta, gridDim.x)) {
    if (tid == 0) a.scratch.splits[cta].parts = 0;
    return;
  }
  const int G = sh.G;
  bool more;
  do {
    const Share& t = w.at;
    const int row0 = t.row_tile * ROWS, rows = min(ROWS, t.n * G - row0);
    const int total = t.ctx + t.n;
    const int* table = a.page_table + (size_t)t.seq * a.pt_stride;
    __syncthreads();
    for (int i = tid; i < ROWS * (D / 4); i += THREADS) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows) {
        const int rr = row0 + r;
        v = load4((const T*)a.q + (size_t)(t.first + rr / G) * a.q_stride + (size_t)(t.head * G + rr % G) * D + d);
      }
      *reinterpret_cast<float4*>(qs + r * LD + d) = v;
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
    for (int kt = t.kt_begin; kt < t.kt_end; ++kt) {
      const int key0 = kt * KEYS;
      __syncthreads();
      if (tid < KEYS) {
        const int key = key0 + tid;
        long at = -1;
        const bool wanted = key < total && (sh.window <= 0 || key > t.ctx - sh.window);
        if (wanted) {
          const int page = key / a.page_size < a.pt_stride ? table[key / a.page_size] : -1;
          if (page >= 0 && page < a.num_pages)
            at = ((long)page * sh.KVH + t.head) * a.page_size + key % a.page_size;
          else
            atomicOr(a.err, DSP_ERR_BAD_PAGE);
        }
        slot_of_key[tid] = at;
      }
      __syncthreads();
      for (int i = tid; i < KEYS * (D / 4); i += THREADS) {
        const int j = i / (D / 4), d = i % (D / 4) * 4;
        const long at = slot_of_key[j];
        float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
        if (at >= 0) {
          k = load4((const T*)a.k_pool + at * D + d);
          v = load4((const T*)a.v_pool + at * D + d);
        }
        *reinterpret_cast<float4*>(ks + j * LD + d) = k;
        *reinterpret_cast<float4*>(vs + j * LD + d) = v;
      }
      __syncthreads();
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
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * alpha + sum;
        m[i] = m_new;
#pragma unroll
        for (int d = 0; d < 4 * DJ; ++d) acc[i][d] *= alpha;
      }
      __syncwarp();  // a row's weights are written and read by the same half warp
      for (int j = 0; j < KEYS; ++j) {
        float e[RI];
#pragma unroll
        for (int i = 0; i < RI; ++i) e[i] = ps[(ty + i * 16) * LP + j];
#pragma unroll
        for (int c = 0; c < DJ; ++c) {
          if (c * 64 + tx * 4 < D) {
            const float4 v = *reinterpret_cast<const float4*>(vs + j * LD + c * 64 + tx * 4);
#pragma unroll
            for (int i = 0; i < RI; ++i) {
              // a hidden key's value, whatever it is, is not part of the sum
              if (e[i] == 0.f) continue;
              acc[i][4 * c] = fmaf(e[i], v.x, acc[i][4 * c]);
              acc[i][4 * c + 1] = fmaf(e[i], v.y, acc[i][4 * c + 1]);
              acc[i][4 * c + 2] = fmaf(e[i], v.z, acc[i][4 * c + 2]);
              acc[i][4 * c + 3] = fmaf(e[i], v.w, acc[i][4 * c + 3]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = ty + i * 16;
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
    const Split split = w.split(sh, cta);
    more = w.next(sh, cta);
    if (!more && tid == 0) a.scratch.splits[cta] = split;
  } while (more);
}

// Every block makes out which CTAs began an item that others share (one read of the list, a thread each), and the warps of the
// whole grid take those items' rows in turn.  A row's partial results are asked for eight at a time, maxima, sums and outputs
// together: two latencies stand between the wait and the store.
constexpr int COMBINE_THREADS = 256, COMBINE_WARPS = COMBINE_THREADS / 32, COMBINE_BLOCKS_PER_SM = 4;
template <typename T>
__global__ void __launch_bounds__(COMBINE_THREADS, COMBINE_BLOCKS_PER_SM)
tree_combine_kernel(const TreeScratch scratch, T* __restrict__ out, long out_stride, int G, int D, int R, int ctas) {
  __shared__ int items[COMBINE_THREADS];  // CTAs that began one
  __shared__ int of_warp[COMBINE_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  for (int c0 = 0; c0 < ctas; c0 += COMBINE_THREADS) {
    const bool has = c0 + tid < ctas && scratch.splits[c0 + tid].parts > 0;
    // the same list in every block: in the order of the CTAs
    const uint32_t those = __ballot_sync(0xffffffffu, has);
    __syncthreads();
    if (lane == 0) of_warp[warp] = __popc(those);
    __syncthreads();
    int before = 0, n_items = 0;
#pragma unroll
    for (int w = 0; w < COMBINE_WARPS; ++w) {
      before += w < warp ? of_warp[w] : 0;
      n_items += of_warp[w];
    }
    if (has) items[before + __popc(those & ((1u << lane) - 1u))] = c0 + tid;
    __syncthreads();
    for (int i = blockIdx.x * COMBINE_WARPS + warp; i < n_items * R; i += gridDim.x * COMBINE_WARPS) {
      // neighbouring warps take neighbouring rows
      const int c = items[i / R], r = i % R;
      const Split x = scratch.splits[c];
      if (r >= x.rows) continue;
      const float2* ml = reinterpret_cast<const float2*>(scratch.part_ml);
      auto row_of = [&](int k) -> size_t { return (k == 0 ? 2 * (size_t)c + 1 : 2 * (size_t)(c + k)) * R + r; };  // of the k-th part
      const int rr = x.row0 + r;
      T* dst = out + (size_t)(x.first + rr / G) * out_stride + (size_t)(x.head * G + rr % G) * D;
      for (int d = lane * 4; d < D; d += 128) {
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < x.parts; k0 += 8) {
          float4 v[8];
          float2 p[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const size_t row = row_of(min(k0 + k, x.parts - 1));
            p[k] = ml[row];
            v[k] = load4(scratch.part_o + row * D + d);
          }
          float top = M;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (k0 + k >= x.parts) p[k] = make_float2(-INFINITY, 0.f);
            top = fmaxf(top, p[k].x);
          }
          if (top == -INFINITY) continue;
          const float w0 = exp2f(M - top);
          L *= w0;
          acc = make_float4(acc.x * w0, acc.y * w0, acc.z * w0, acc.w * w0);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (p[k].x == -INFINITY) continue;  // a part that saw no key
            const float w = exp2f(p[k].x - top);
            L = fmaf(w, p[k].y, L);
            acc = make_float4(fmaf(w, v[k].x, acc.x), fmaf(w, v[k].y, acc.y), fmaf(w, v[k].z, acc.z), fmaf(w, v[k].w, acc.w));
          }
          M = top;
        }
        const float inv = L > 0.f ? 1.f / L : 0.f;
        store4(dst + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      }
    }
  }
}

template <typename T>
int launch(const Args& a, int ctas, cudaStream_t stream) {
  const size_t smem = (size_t)((ROWS + 2 * KEYS) * (a.D + 4) + ROWS * LP) * sizeof(float);
  auto go = [&](auto kernel) -> int {
    DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    DSP_CUDA(launch_plain(kernel, dim3(ctas), dim3(THREADS), smem, stream, a));
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

// The same for kernels that live in other libraries.
extern "C" int dsp_tree_combine(const TreeScratch* scratch, void* out, long out_stride, int G, int D, int rows_per_tile,
                                int ctas, int dtype, cudaStream_t stream) {
  return tree_combine(*scratch, out, out_stride, G, D, rows_per_tile, ctas, dtype, stream) == cudaSuccess ? 0 : 1;
}

// What the Python side packs, in this order (ops/tree.py).
struct DspTreeAttention {
  const void *q, *k_pool, *v_pool;
  const int *page_table, *ctx_len, *node_start, *depth;
  const unsigned long long* visible;
  void* out;
  float* scratch;
  long q_stride, out_stride, pt_stride, words, S, H, KVH, D, page_size, num_pages, window, dtype, ctas;
  double scale;
};

extern "C" int dsp_tree_attention(const DspTreeAttention* p, cudaStream_t stream) {
  if (p->S == 0) return 0;
  DSP_REQUIRE(p->S > 0 && p->KVH > 0 && p->H > 0 && p->H % p->KVH == 0, "dsp_tree_attention: %ld heads on %ld key/value heads",
              p->H, p->KVH);
  DSP_REQUIRE(p->D % 8 == 0 && p->D >= 8 && p->D <= 256, "dsp_tree_attention: head size %ld (a multiple of 8 up to 256)", p->D);
  DSP_REQUIRE(p->dtype == DSP_F32 || p->dtype == DSP_BF16, "dsp_tree_attention: unknown dtype %ld", p->dtype);
  DSP_REQUIRE(p->ctas >= 1 && p->page_size >= 1 && p->num_pages >= 0 && p->words >= 1, "dsp_tree_attention: bad sizes");
  const uintptr_t bits = (uintptr_t)p->q | (uintptr_t)p->k_pool | (uintptr_t)p->v_pool | (uintptr_t)p->out;
  DSP_REQUIRE(bits % 16 == 0 && p->q_stride % 8 == 0 && p->out_stride % 8 == 0,
              "dsp_tree_attention: rows must begin on 16 bytes");
  Args a = {};
  a.sh.node_start = p->node_start;
  a.sh.ctx_len = p->ctx_len;
  a.sh.S = (int)p->S;
  a.sh.KVH = (int)p->KVH;
  a.sh.G = (int)(p->H / p->KVH);
  a.sh.rows_per_tile = ROWS;
  a.sh.keys_per_tile = KEYS;
  a.sh.window = (int)p->window;
  a.sh.min_units = 1;
  a.q = p->q;
  a.k_pool = p->k_pool;
  a.v_pool = p->v_pool;
  a.page_table = p->page_table;
  a.depth = p->depth;
  a.visible = p->visible;
  a.out = p->out;
  a.scratch = tree_scratch(p->scratch, p->ctas, ROWS, p->D);
  a.q_stride = p->q_stride;
  a.out_stride = p->out_stride;
  a.pt_stride = (int)p->pt_stride;
  a.words = (int)p->words;
  a.D = (int)p->D;
  a.page_size = (int)p->page_size;
  a.num_pages = (int)p->num_pages;
  a.scale = (float)p->scale;
  a.err = dsp_device_error_ptr();
  DSP_REQUIRE(a.err != nullptr, "dsp_tree_attention: no device error word");
  const int rc = p->dtype == DSP_F32 ? launch<float>(a, (int)p->ctas, stream) : launch<bf16>(a, (int)p->ctas, stream);
  if (rc != 0) return rc;
  DSP_CUDA(tree_combine(a.scratch, a.out, a.out_stride, a.sh.G, a.D, ROWS, (int)p->ctas, (int)p->dtype, stream));
  DSP_CHECK_LAUNCH("dsp_tree_attention");
  return 0;
}
