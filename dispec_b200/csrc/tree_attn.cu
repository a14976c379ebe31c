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
  float *part_o, *part_ml;
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
  if (!w.begin(sh, cta, gridDim.x)) return;
  const int G = sh.G;
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
          store4(a.part_o + ((size_t)t.slot * ROWS + r) * D + d, v);
        else
          store4((T*)a.out + (size_t)(t.first + rr / G) * a.out_stride + (size_t)(t.head * G + rr % G) * D + d, v);
      }
      if (t.slot >= 0 && tx == 0)
        reinterpret_cast<float2*>(a.part_ml)[(size_t)t.slot * ROWS + r] = make_float2(m[i] * 1.4426950408889634f, l[i]);
    }
  } while (w.next(sh, cta));
}

// Block (c, y): the item that begins in CTA c and ends in a later one, if there is one; four of its rows, one a warp.  Which
// item that is does not depend on the kernel in front, so it is found out before the wait.  A lane holds the weights
// of up to 32 partial results, and the outputs of eight are asked for together.
template <typename T>
__global__ void __launch_bounds__(128)
tree_combine_kernel(const Shape sh, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                    T* __restrict__ out, long out_stride, int D, int ctas) {
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  // last unit of CTA c
  const Found f = find_unit(sh, ctas, [&](const Found& g) {
    const long last = min((long)g.total, (long)g.chunk * (c + 1)) - 1;
    return last + 1 >= g.total ? g.total : (int)last;  // (nothing follows the last CTA with work)
  });
  bool mine = f.seq >= 0;
  int c_end = 0, head = 0, row0 = 0, rows = 0;
  Tree t = {};
  if (mine) {
    t = load_tree(sh, f.seq);
    const int last = f.chunk * (c + 1) - 1;
    head = (last - f.start) / t.key_tiles;
    const int begin = f.start + head * t.key_tiles, end = begin + t.key_tiles;
    mine = end != last + 1 && begin >= f.chunk * c;  // it goes on, and began here
    c_end = (end - 1) / f.chunk;
    row0 = f.row_tile * sh.rows_per_tile;
    rows = min(sh.rows_per_tile, t.n * sh.G - row0);
  }
  const int r = blockIdx.y * 4 + warp;
  pdl_wait();
  if (!mine || r >= rows) return;
  const float2* ml = reinterpret_cast<const float2*>(part_ml);
  const int R = sh.rows_per_tile, parts = c_end - c + 1;
  auto slot = [&](int k) -> size_t { return k == 0 ? 2 * (size_t)c + 1 : 2 * (size_t)(c + k); };  // of the k-th part
  float M = -INFINITY, L = 0.f;
  float2 mine_ml = make_float2(-INFINITY, 0.f);
  for (int k = lane; k < parts; k += 32) {
    const float2 v = ml[slot(k) * R + r];
    if (k < 32) mine_ml = v;
    M = fmaxf(M, v.x);
  }
  M = warp_max(M);
  for (int k = lane; k < parts; k += 32) {
    const float2 v = k < 32 ? mine_ml : ml[slot(k) * R + r];
    if (v.x != -INFINITY) L += v.y * exp2f(v.x - M);
  }
  L = warp_sum(L);
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const int rr = row0 + r;
  T* dst = out + (size_t)(t.first + rr / sh.G) * out_stride + (size_t)(head * sh.G + rr % sh.G) * D;
  for (int d0 = 0; d0 < D; d0 += 128) {  // the same trips for a whole warp (shuffles)
    const int d = d0 + lane * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < parts; k0 += 8) {
      float4 v[8];
      float wk[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int part = k0 + k;
        float m = -INFINITY;
        if (part < 32)
          m = __shfl_sync(0xffffffffu, mine_ml.x, part);
        else if (part < parts)
          m = ml[slot(part) * R + r].x;
        wk[k] = part < parts && m != -INFINITY ? exp2f(m - M) : 0.f;
        v[k] = wk[k] != 0.f && d < D ? load4(part_o + (slot(part) * R + r) * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        acc.x = fmaf(wk[k], v[k].x, acc.x);
        acc.y = fmaf(wk[k], v[k].y, acc.y);
        acc.z = fmaf(wk[k], v[k].z, acc.z);
        acc.w = fmaf(wk[k], v[k].w, acc.w);
      }
    }
    if (d < D) store4(dst + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
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

cudaError_t tree_combine(const tree::Shape& sh, const float* part_o, const float* part_ml, void* out, long out_stride,
                         int D, int ctas, int dtype, cudaStream_t stream) {
  const dim3 grid(ctas, (sh.rows_per_tile + 3) / 4);
  return dtype == DSP_F32
             ? launch_pdl(tree_combine_kernel<float>, grid, dim3(128), 0, stream, sh, part_o, part_ml, (float*)out, out_stride, D, ctas)
             : launch_pdl(tree_combine_kernel<bf16>, grid, dim3(128), 0, stream, sh, part_o, part_ml, (bf16*)out, out_stride, D, ctas);
}

// The same for kernels that live in other libraries.
extern "C" int dsp_tree_combine(const tree::Shape* sh, const float* part_o, const float* part_ml, void* out, long out_stride,
                                int D, int ctas, int dtype, cudaStream_t stream) {
  return tree_combine(*sh, part_o, part_ml, out, out_stride, D, ctas, dtype, stream) == cudaSuccess ? 0 : 1;
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
  a.part_o = p->scratch;
  a.part_ml = p->scratch + 2 * p->ctas * ROWS * p->D;
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
  DSP_CUDA(tree_combine(a.sh, a.part_o, a.part_ml, a.out, a.out_stride, a.D, (int)p->ctas, (int)p->dtype, stream));
  DSP_CHECK_LAUNCH("dsp_tree_attention");
  return 0;
}
