// Verification of drafted trees: the walk from a tree's root along accepted drafts, and the token drawn where it ends.
//
// The logits of node i's row give the target's distribution of the token behind node i.  It is held in whole numbers, the
// likeliest token's mass being 2^40:
//     m_v = floor(2^40 exp(x_v - max x)),  x = logits / temperature
// (temperature 0: all of it on the largest logit, ties to the lowest index).  Sums of whole numbers do not depend on their
// order, so neither does any decision.  Standing at node cur with the masses m, R = sum m, the children of cur are tried
// in index order.  Child c with token t, its uniform number u and q the distribution that cur's children were drawn from:
//     taken   iff  (u q_t) R < m_t            (without draft probabilities q_t = 1)
//     refused:     m_v <- max(0, m_v - floor(q_v R)), without draft probabilities m_t <- 0
// and where nothing would be left m stays.  A refused draft leaves the masses in proportion to max(0, p - q), so that the
// accepted tokens and the drawn one together are distributed as the target's own samples.  Where no child is taken, the
// token is the first v whose masses up to v exceed min(R - 1, floor(draw R)).  NaN counts as -inf; a row without a finite
// or infinite largest logit gives token 0.
//
// A cluster of up to 16 CTAs works on one tree and reads only the rows of the nodes that the walk comes to, each of them
// once: every CTA keeps its share of the row in shared memory, first as scaled logits, then as exponentials, and the CTAs
// exchange the largest logit and the sums of masses through each other's shared memory (one cluster barrier each).  The
// tests of a node's children need R and a few numbers that are read while the row arrives; every CTA makes them for itself, with the same result.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {
constexpr int THREADS = 512, WARPS = THREADS / 32, MAX_CTAS = 16, MAX_NODES = 1024;
constexpr int SHARE = 24 * 1024;      // logits of a row in a CTA's shared memory, two CTAs an SM
constexpr int MAX_VOCAB = 1 << 19;    // 32,768 logits in each of 16 CTAs
typedef long long mass_t;
constexpr mass_t ONE = (mass_t)1 << 40;

struct Args {
  const void* logits;
  const float* draft;
  const int *tokens, *parents, *node_start;
  const float *temperature, *uniforms, *draws;
  int *path, *count, *token;
  long ld, ldq;
  int V, share, max_nodes;
  int* err;
};

__device__ __forceinline__ mass_t warp_sum_mass(mass_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float scale_logit(float l, float temp) {
  return isnan(l) ? -INFINITY : temp > 0.f ? __fdiv_rn(l, temp) : l;
}
__device__ __forceinline__ float exponential(float x, float top) { return x == top ? 1.f : expf(x - top); }
__device__ __forceinline__ mass_t mass_of(float e) { return (mass_t)(e * 1099511627776.f); }

// One exchange: every CTA of the cluster tells every other one a number.
struct Mailbox {
  float value[2][MAX_CTAS];
  mass_t mass[2][MAX_CTAS];
};

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(THREADS)
tree_verify_kernel(const Args a) {
  extern __shared__ float xs[];  // [share] this CTA's part of the row
  __shared__ Mailbox box;
  __shared__ int parents[MAX_NODES];
  __shared__ float cand_x[MAX_NODES], cand_q[MAX_NODES], cand_u[MAX_NODES];  // of the children of the present node
  __shared__ int cand_t[MAX_NODES];
  __shared__ int gone[MAX_NODES];    // refused tokens, without draft probabilities
  __shared__ float left[MAX_NODES];  // R at each refusal, with them
  __shared__ float warp_value[WARPS];
  __shared__ mass_t warp_mass[WARPS];
  __shared__ mass_t cta_mass[MAX_CTAS];  // the masses of every CTA's part
  __shared__ mass_t total;               // R
  __shared__ int decided, refused, first_top;

  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int s = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (ctas > 1) cluster.sync();  // every CTA of the cluster is there before another one writes to it
  pdl_wait();
  pdl_launch_dependents();
  const int first = a.node_start[s], n = min(a.node_start[s + 1] - first, a.max_nodes);
  int* path = a.path + (size_t)s * a.max_nodes;
  if (rank == 0)
    for (int i = tid; i < a.max_nodes; i += THREADS) path[i] = i == 0 && n > 0 ? 0 : -1;
  if (n <= 0) {  // (the whole cluster leaves)
    if (rank == 0 && tid == 0) {
      a.count[s] = 0;
      a.token[s] = -1;
    }
    return;
  }
  for (int i = tid; i < n; i += THREADS) parents[i] = a.parents[first + i];
  const float temp = a.temperature[s];
  const int begin = min(a.V, rank * a.share), end = min(a.V, begin + a.share), mine = end - begin;
  int turn = 0;

  // the largest of all threads' values in the cluster
  auto cluster_max = [&](float v) -> float {
    v = warp_max(v);
    __syncthreads();
    if (lane == 0) warp_value[warp] = v;
    __syncthreads();
    v = lane < WARPS ? warp_value[lane] : -INFINITY;
    v = warp_max(v);
    if (ctas == 1) return v;
    if (tid < ctas) cluster.map_shared_rank(&box, tid)->value[turn][rank] = v;
    cluster.sync();
    v = lane < ctas ? box.value[turn][lane] : -INFINITY;
    turn ^= 1;
    return warp_max(v);
  };
  // the sum of all threads' masses in the cluster; cta_mass has every CTA's afterwards (behind the next block barrier)
  auto cluster_sum = [&](mass_t v) -> mass_t {
    v = warp_sum_mass(v);
    __syncthreads();
    if (lane == 0) warp_mass[warp] = v;
    __syncthreads();
    v = warp_sum_mass(lane < WARPS ? warp_mass[lane] : 0);
    if (ctas > 1) {
      if (tid < ctas) cluster.map_shared_rank(&box, tid)->mass[turn][rank] = v;
      cluster.sync();
      const mass_t each = lane < ctas ? box.mass[turn][lane] : 0;
      if (tid < ctas) cta_mass[tid] = each;
      turn ^= 1;
      return warp_sum_mass(each);
    }
    if (tid == 0) cta_mass[0] = v;
    return v;
  };

  int cur = 0, count = 1;
  for (;;) {
    // ---- the row of node cur
    const T* row = (const T*)a.logits + (size_t)(first + cur) * a.ld;
    const float* q = DRAFT ? a.draft + (size_t)(first + cur) * a.ldq : nullptr;
    __syncthreads();  // parents are there; nobody reads the last row any more
    for (int i = cur + 1 + tid; i < n; i += THREADS) {
      if (parents[i] != cur) continue;
      const int t = a.tokens[first + i];
      const bool known = t >= 0 && t < a.V;
      if (!known) atomicOr(a.err, DSP_ERR_BAD_TOKEN);
      cand_t[i] = known ? t : -1;
      cand_u[i] = a.uniforms[first + i];
      cand_x[i] = known ? scale_logit(to_f32(row[t]), temp) : 0.f;
      cand_q[i] = DRAFT && known ? q[t] : 1.f;
    }
    float top = -INFINITY;
    {
      constexpr int N = 16 / sizeof(T);
      const T* src = row + begin;
      int done = 0;
      if (((uintptr_t)src & 15) == 0) {  // (a share is a multiple of 16 bytes)
        const int pieces = mine / N;
        constexpr int AHEAD = 5;  // requests of a thread under way: a share of 151,936 / 16 logits at once
        for (int i0 = tid; i0 < pieces; i0 += AHEAD * THREADS) {
          uint4 v[AHEAD];
#pragma unroll
          for (int k = 0; k < AHEAD; ++k)
            if (i0 + k * THREADS < pieces) v[k] = __ldg(reinterpret_cast<const uint4*>(src) + i0 + k * THREADS);
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + k * THREADS;
            if (i >= pieces) continue;
            const T* l = reinterpret_cast<const T*>(&v[k]);
#pragma unroll
            for (int c = 0; c < N; ++c) {
              const float x = scale_logit(to_f32(l[c]), temp);
              xs[i * N + c] = x;
              top = fmaxf(top, x);
            }
          }
        }
        done = pieces * N;
      }
#pragma unroll 4
      for (int i = done + tid; i < mine; i += THREADS) {
        const float x = scale_logit(to_f32(src[i]), temp);
        xs[i] = x;
        top = fmaxf(top, x);
      }
    }
    top = cluster_max(top);
    const bool alone = !(temp > 0.f) || top == -INFINITY;  // all the mass on the lowest index of `top`
    if (alone) {
      int low = a.V;
      for (int i = tid; i < mine; i += THREADS)
        if (xs[i] == top) low = min(low, begin + i);
      first_top = (int)-cluster_max((float)-low);  // (whole numbers up to 2^24 are exact)
      __syncthreads();
      const int at = first_top;
      for (int i = tid; i < mine; i += THREADS) xs[i] = begin + i == at ? 1.f : 0.f;
      if (tid < ctas) cta_mass[tid] = at >= tid * a.share && at < (tid + 1) * a.share ? ONE : 0;
      if (tid == 0) total = ONE;
    } else {
      mass_t sum = 0;
#pragma unroll 4
      for (int i = tid; i < mine; i += THREADS) {
        const float e = exponential(xs[i], top);
        xs[i] = e;
        sum += mass_of(e);
      }
      sum = cluster_sum(sum);
      if (tid == 0) total = sum;
    }
    if (tid == 0) refused = 0;
    __syncthreads();

    // ---- its children, in the order of their numbers
    int next = cur + 1;
    for (;;) {
      if (warp == 0) {
        mass_t R = total;
        int found = 0, nr = refused;
        for (int i0 = next & ~31; i0 < n && found == 0; i0 += 32) {
          const int me = i0 + lane;
          uint32_t todo = __ballot_sync(0xffffffffu, me >= next && me < n && parents[me] == cur);
          while (todo != 0u && found == 0) {
            const int i = i0 + __ffs(todo) - 1;
            todo &= todo - 1;
            const int t = cand_t[i];
            if (t < 0) continue;
            const float e = alone ? (t == first_top ? 1.f : 0.f) : exponential(cand_x[i], top);
            mass_t m = mass_of(e);
            if (DRAFT) {
              for (int k = 0; k < nr; ++k) m = max((mass_t)0, m - (mass_t)__fmul_rn(cand_q[i], left[k]));
              if (__fmul_rn(__fmul_rn(cand_u[i], cand_q[i]), (float)R) < (float)m)
                found = i;
              else
                found = -i;  // refused: the masses have to be summed again
            } else {
              bool was = false;  // refused before: no mass
              for (int k = lane; k < nr; k += 32) was |= gone[k] == t;
              if (__any_sync(0xffffffffu, was)) m = 0;
              if (__fmul_rn(cand_u[i], (float)R) < (float)m) {
                found = i;
              } else if (m > 0 && R > m) {
                R -= m;
                if (lane == 0) {
                  gone[nr] = t;
                  cta_mass[t / a.share] -= m;
                }
                ++nr;
                __syncwarp();
              }
            }
          }
        }
        if (lane == 0) {
          decided = found;
          if (!DRAFT) {
            total = R;
            refused = nr;
          } else if (found < 0) {
            left[nr] = (float)R;
          }
        }
      }
      __syncthreads();
      if (!DRAFT || decided >= 0) break;
      const int nr = refused + 1;
      mass_t sum = 0;
#pragma unroll 4
      for (int i = tid; i < mine; i += THREADS) {
        mass_t m = mass_of(xs[i]);
        const float qv = q[begin + i];
        for (int k = 0; k < nr; ++k) m = max((mass_t)0, m - (mass_t)__fmul_rn(qv, left[k]));
        sum += m;
      }
      next = -decided + 1;
      // (where nothing would be left, the masses and every CTA's sum stay)
      const mass_t kept = tid < ctas ? cta_mass[tid] : 0;
      const mass_t rest = cluster_sum(sum);
      if (rest == 0 && tid < ctas) cta_mass[tid] = kept;
      if (rest > 0 && tid == 0) {
        total = rest;
        refused = nr;
      }
      __syncthreads();
    }
    if (decided <= 0) {
      // ---- no child was taken: the draw, by the CTA whose part holds the mass it aims at
      const mass_t R = total, aim = max((mass_t)0, min((mass_t)__fmul_rn(a.draws[s], (float)R), R - 1));
      mass_t before = 0;
      for (int r = 0; r < rank; ++r) before += cta_mass[r];
      if (before <= aim && aim < before + cta_mass[rank]) {
        const int nr = refused;
        auto mass_at = [&](int i) -> mass_t {
          mass_t m = mass_of(xs[i]);
          if (DRAFT) {
            const float qv = nr > 0 ? q[begin + i] : 0.f;
            for (int k = 0; k < nr; ++k) m = max((mass_t)0, m - (mass_t)__fmul_rn(qv, left[k]));
          } else {
            for (int k = 0; k < nr; ++k)
              if (gone[k] == begin + i) m = 0;
          }
          return m;
        };
        // every warp has a run of neighbouring tokens, 32 at a time
        const int per = (mine + WARPS * 32 - 1) / (WARPS * 32) * 32, w0 = min(mine, warp * per), w1 = min(mine, w0 + per);
        mass_t sum = 0;
#pragma unroll 4
        for (int i = w0 + lane; i < w1; i += 32) sum += mass_at(i);
        sum = warp_sum_mass(sum);
        if (lane == 0) warp_mass[warp] = sum;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before += warp_mass[w];
        if (before <= aim && aim < before + sum) {
          for (int i0 = w0;; i0 += 32) {
            mass_t upto = i0 + lane < w1 ? mass_at(i0 + lane) : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const mass_t up = __shfl_up_sync(0xffffffffu, upto, o);
              if (lane >= o) upto += up;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + upto > aim);
            if (past != 0u) {
              if (lane == 0) a.token[s] = begin + i0 + __ffs(past) - 1;
              break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
          }
        }
      }
      if (rank == 0 && tid == 0) a.count[s] = count;
      break;
    }
    cur = decided;
    if (rank == 0 && tid == 0) path[count] = cur;
    ++count;
  }
  // (nobody writes to another CTA after the last exchange, whose barrier all of them passed)
}

template <typename T, bool DRAFT>
int launch(const Args& a, int S, int ctas, cudaStream_t stream) {
  auto kernel = tree_verify_kernel<T, DRAFT>;
  const size_t smem = (size_t)a.share * sizeof(float);
  prefer_max_shared(reinterpret_cast<const void*>(kernel));
  DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  if (ctas > 8) DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(S * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  DSP_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return 0;
}
}  // namespace

// What the Python side packs, in this order (ops/tree.py).
struct DspTreeVerify {
  const void* logits;
  const float* draft;
  const int *tokens, *parents, *node_start;
  const float *temperature, *uniforms, *draws;
  int *path, *count, *token;
  long ld, ldq, S, V, max_nodes, dtype;
};

extern "C" int dsp_tree_verify(const DspTreeVerify* p, cudaStream_t stream) {
  if (p->S == 0) return 0;
  DSP_REQUIRE(p->S > 0 && p->V > 0 && p->V <= MAX_VOCAB, "dsp_tree_verify: a vocabulary of %ld (at most 2^19)", p->V);
  DSP_REQUIRE(p->max_nodes > 0 && p->max_nodes <= MAX_NODES, "dsp_tree_verify: max_nodes=%ld", p->max_nodes);
  DSP_REQUIRE(p->dtype == DSP_F32 || p->dtype == DSP_BF16, "dsp_tree_verify: unknown dtype %ld", p->dtype);
  Args a = {};
  a.logits = p->logits;
  a.draft = p->draft;
  a.tokens = p->tokens;
  a.parents = p->parents;
  a.node_start = p->node_start;
  a.temperature = p->temperature;
  a.uniforms = p->uniforms;
  a.draws = p->draws;
  a.path = p->path;
  a.count = p->count;
  a.token = p->token;
  a.ld = p->ld;
  a.ldq = p->ldq;
  a.V = (int)p->V;
  a.max_nodes = (int)p->max_nodes;
  a.err = dsp_device_error_ptr();
  DSP_REQUIRE(a.err != nullptr, "dsp_tree_verify: no device error word");
  // CTAs a tree: as many as keep the device's SMs busy with the trees there are, at least 2,048 logits each, and so many
  // that a share fits
  const int sms = dsp_num_sms();
  int ctas = 1;
  while (ctas < MAX_CTAS && ((p->V + ctas - 1) / ctas > SHARE || (ctas * 2 * 2048 <= p->V && ctas * 2 * p->S <= 2 * sms))) ctas *= 2;
  a.share = (int)(((p->V + ctas - 1) / ctas + 7) / 8 * 8);
  const int S = (int)p->S;
  const int rc = p->dtype == DSP_F32 ? (a.draft ? launch<float, true>(a, S, ctas, stream) : launch<float, false>(a, S, ctas, stream))
                                     : (a.draft ? launch<bf16, true>(a, S, ctas, stream) : launch<bf16, false>(a, S, ctas, stream));
  if (rc != 0) return rc;
  DSP_CHECK_LAUNCH("dsp_tree_verify");
  return 0;
}
