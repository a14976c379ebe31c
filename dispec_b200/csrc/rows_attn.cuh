// Attention of rows over the paged cache in 32-bit arithmetic.  What the rows are, how the work is cut and what a row sees is said by
// a type `Work` (TreeWork in tree_schedule.cuh, SharedWork in shared_schedule.cuh).
//
// A block holds 32 rows and walks key tiles of 64, queries, keys and values as floats in shared memory: thread
// (ty, tx) of 16 x 16 owns rows ty, ty + 16 and keys tx + 16 j of the scores, and of the result the same rows and
// the dimensions 4 tx .. 4 tx + 3 of each 64.  Maximum and sum of a row are exchanged between its 16 threads by
// shuffles.  Multiply-adds and the reads from shared memory that feed them (5 for every 16, two cycles each) bound it: for 8
// trees of 32 nodes behind 4,000 tokens, 12 heads of 128 on 2, 32-bit, 223 us, 21 TFLOP/s.  Up to head size 128 two blocks
// share an SM, so that one's copies and softmax run beside the other's products (513 us with one, whose rows were copied
// between barriers); keys and values come while the tile before is still being used.
#pragma once
#include <type_traits>

#include "rows_schedule.cuh"

namespace {

constexpr int ROW_SHIFT = ROW_SHIFT_32BIT, ROWS = 1 << ROW_SHIFT, KEYS = KEYS_PER_TILE, TX = 16, THREADS = 256, RI = ROWS / 16, KJ = KEYS / TX, LP = KEYS + 4;

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
template <typename Work, typename T, int DJ>
__global__ void __launch_bounds__(THREADS, DJ == 4 ? 1 : 2)
rows_attn_kernel(const typename Work::Args a) {
  typedef typename Work::Share Share;
  extern __shared__ float smem[];
  const int D = a.D, LD = D + 4, tid = threadIdx.x, tx = tid % TX, ty = tid / TX;
  float* qs = smem;              // [ROWS][LD]
  float* ks = qs + ROWS * LD;    // [KEYS][LD]
  float* vs = ks + KEYS * LD;    // [KEYS][LD]
  float* ps = vs + KEYS * LD;    // [ROWS][LP]
  __shared__ long slots_of_keys[2][KEYS];  // of this key tile and the coming one
  const auto& sh = a.sh;
  __shared__ typename Work::Plan plan;
  typename Work::Walk w;
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: what comes next may look at the inputs before it waits)
  Work::make_plan(sh, plan, blockIdx.x, gridDim.x);
  if (!Work::begin(w, sh, plan, blockIdx.x, gridDim.x)) {
    if (tid == 0) Work::note_none(a, w.cta);
    return;
  }
  const int G = sh.G;
  bool more;
  do {
    const Share& t = w.at;
    const int row0 = t.row_tile * ROWS, rows = min(ROWS, t.n * G - row0);
    const int first_key = Work::key_begin(sh, t), total = Work::key_end(t);
    const int* table = a.page_table + (size_t)t.seq * a.pt_stride;
    auto find_keys = [&](int kt) {
      const int key = kt * KEYS + tid;
      long at = -1;
      if (key < total && key >= first_key) {
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
    int node[RI];
    typename Work::Row seen_by[RI];
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = ty + i * 16;
      node[i] = r < rows ? t.first + (row0 + r) / G : -1;
      seen_by[i] = Work::row(a, t, node[i] >= 0 ? node[i] : t.first);
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
          const bool seen = node[i] >= 0 && slot_of_key[tx + j * TX] >= 0 && Work::sees(a, t, seen_by[i], key);
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
      // (a page that is not there has values of zero)
      if (Work::whole(sh, t, key0))
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
      const float inv = t.slot >= 0 || Work::ROW_PARTS ? 1.f : l[i] > 0.f ? 1.f / l[i] : 0.f;
#pragma unroll
      for (int c = 0; c < DJ; ++c) {
        const int d = c * 64 + tx * 4;
        if (d >= D) continue;
        const float4 v = make_float4(acc[i][4 * c] * inv, acc[i][4 * c + 1] * inv, acc[i][4 * c + 2] * inv,
                                     acc[i][4 * c + 3] * inv);
        if (t.slot >= 0)
          store4(a.scratch.part_o + ((size_t)t.slot * ROWS + r) * D + d, v);
        else if constexpr (Work::ROW_PARTS)
          store4(a.scratch.rows_o + Work::row_part(sh, t, rr) * D + d, v);
        else
          store4((T*)a.out + (size_t)(t.first + rr / G) * a.out_stride + (size_t)(t.head * G + rr % G) * D + d, v);
      }
      if (tx == 0) {
        const float2 ml = make_float2(m[i] * 1.4426950408889634f, l[i]);
        if (t.slot >= 0) {
          reinterpret_cast<float2*>(a.scratch.part_ml)[(size_t)t.slot * ROWS + r] = ml;
        } else {
          if constexpr (Work::ROW_PARTS) reinterpret_cast<float2*>(a.scratch.rows_ml)[Work::row_part(sh, t, rr)] = ml;
        }
      }
    }
    const auto split = w.split(sh);
    more = w.next(sh);
    if (tid == 0) Work::note(a, w.cta, split, more);
  } while (more);
}

template <typename Work, typename T>
int launch_rows_attn(const typename Work::Args& a, cudaStream_t stream) {
  const size_t smem = (size_t)((ROWS + 2 * KEYS) * (a.D + 4) + ROWS * LP) * sizeof(float);
  auto go = [&](auto kernel) -> int {
    DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    DSP_CUDA(launch_pdl(kernel, dim3((unsigned)a.ctas), dim3(THREADS), smem, stream, a));
    return 0;
  };
  return a.D <= 64 ? go(rows_attn_kernel<Work, T, 1>) : a.D <= 128 ? go(rows_attn_kernel<Work, T, 2>) : go(rows_attn_kernel<Work, T, 4>);
}
}  // namespace
