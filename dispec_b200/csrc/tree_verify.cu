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
#include "common.cuh"

namespace {
constexpr int THREADS = 1024;
typedef long long mass_t;

struct Args {
  const void* logits;
  const float* draft;
  const int *tokens, *parents, *node_start;
  const float *temperature, *uniforms, *draws;
  int *path, *count, *token;
  long ld, ldq;
  int V, max_nodes;
  int* err;
};

__device__ __forceinline__ mass_t warp_sum_mass(mass_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a pass over a row needs to know.
template <typename T>
struct Row {
  const T* x;
  const float* q;   // draft probabilities, or null
  float temp, top;  // largest scaled logit
  int first;        // lowest index of it
  bool alone;       // all the mass is on `first`
  int refused;      // refusals so far
  const float* left;  // with draft probabilities: R at each refusal
  const int* gone;    // without: the refused tokens

  __device__ __forceinline__ float scaled(int v) const {
    const float l = to_f32(x[v]);
    return isnan(l) ? -INFINITY : temp > 0.f ? __fdiv_rn(l, temp) : l;
  }
  __device__ __forceinline__ mass_t mass(int v) const {
    mass_t m;
    if (alone) {
      m = v == first ? (mass_t)1 << 40 : 0;
    } else {
      const float s = scaled(v);
      m = s == top ? (mass_t)1 << 40 : (mass_t)(expf(s - top) * 1099511627776.f);
    }
    if (q != nullptr) {
      const float qv = refused > 0 ? q[v] : 0.f;
      for (int k = 0; k < refused; ++k) m = max((mass_t)0, m - (mass_t)__fmul_rn(qv, left[k]));
    } else {
      for (int k = 0; k < refused; ++k)
        if (gone[k] == v) m = 0;
    }
    return m;
  }
};

template <typename T>
__global__ void __launch_bounds__(THREADS)
tree_verify_kernel(const Args a) {
  extern __shared__ int list[];  // [max_nodes] refused tokens, or the R at each refusal
  __shared__ float f_scratch[32];
  __shared__ mass_t m_scratch[32];
  __shared__ int found;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const int first = a.node_start[s], n = min(a.node_start[s + 1] - first, a.max_nodes);
  int* path = a.path + (size_t)s * a.max_nodes;
  for (int i = tid; i < a.max_nodes; i += THREADS) path[i] = -1;
  if (n <= 0) {
    if (tid == 0) {
      a.count[s] = 0;
      a.token[s] = -1;
    }
    return;
  }
  auto sum = [&](mass_t v) -> mass_t {
    v = warp_sum_mass(v);
    __syncthreads();
    if (lane == 0) m_scratch[warp] = v;
    __syncthreads();
    mass_t total = 0;
    for (int w = 0; w < THREADS / 32; ++w) total += m_scratch[w];
    return total;
  };
  Row<T> row;
  row.temp = a.temperature[s];
  row.left = reinterpret_cast<const float*>(list);
  row.gone = list;
  int cur = 0, count = 1;
  mass_t R = 0;
  auto total_of_row = [&]() -> mass_t {
    mass_t v = 0;
    for (int i = tid; i < V; i += THREADS) v += row.mass(i);
    return sum(v);
  };
  auto enter = [&](int node) {
    row.x = (const T*)a.logits + (size_t)(first + node) * a.ld;
    row.q = a.draft ? a.draft + (size_t)(first + node) * a.ldq : nullptr;
    row.refused = 0;
    float top = -INFINITY;
    for (int i = tid; i < V; i += THREADS) top = fmaxf(top, row.scaled(i));
    row.top = block_max(top, f_scratch);
    row.alone = !(row.temp > 0.f) || row.top == -INFINITY;
    int low = V;
    if (row.alone) {
      for (int i = tid; i < V; i += THREADS)
        if (row.scaled(i) == row.top) low = min(low, i);
      if (tid == 0) found = V;
      __syncthreads();
      if (low < V) atomicMin(&found, low);
      __syncthreads();
      low = found;
      __syncthreads();
    }
    row.first = low;
    R = total_of_row();
  };
  __syncthreads();
  if (tid == 0) path[0] = 0;
  enter(0);
  for (int i = 1; i < n; ++i) {
    if (a.parents[first + i] != cur) continue;
    const int t = a.tokens[first + i];
    if (t < 0 || t >= V) {
      if (tid == 0) atomicOr(a.err, DSP_ERR_BAD_TOKEN);
      continue;  // no draft: never taken, nothing to refuse
    }
    const float u = a.uniforms[first + i];
    const float limit = __fmul_rn(row.q ? __fmul_rn(u, row.q[t]) : u, (float)R);
    if (limit < (float)row.mass(t)) {
      cur = i;
      if (tid == 0) path[count] = i;
      ++count;
      enter(i);
      continue;
    }
    __syncthreads();
    if (tid == 0) {
      if (row.q)
        reinterpret_cast<float*>(list)[row.refused] = (float)R;
      else
        list[row.refused] = t;
    }
    __syncthreads();
    ++row.refused;
    const mass_t rest = total_of_row();
    if (rest > 0)
      R = rest;
    else
      --row.refused;
  }
  // the draw: thread t owns a run of neighbouring tokens
  const mass_t aim = max((mass_t)0, min((mass_t)__fmul_rn(a.draws[s], (float)R), R - 1));
  const int per = (V + THREADS - 1) / THREADS, begin = min(V, tid * per), end = min(V, begin + per);
  mass_t mine = 0;
  for (int i = begin; i < end; ++i) mine += row.mass(i);
  mass_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const mass_t up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  __syncthreads();
  if (lane == 31) m_scratch[warp] = upto;
  __syncthreads();
  mass_t before = upto - mine;
  for (int w = 0; w < warp; ++w) before += m_scratch[w];
  if (before <= aim && aim < before + mine) {
    int v = begin;
    for (; v < end; ++v) {
      before += row.mass(v);
      if (before > aim) break;
    }
    a.token[s] = v;
  }
  if (tid == 0) a.count[s] = count;
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
  DSP_REQUIRE(p->S > 0 && p->V > 0 && p->V <= (1 << 22), "dsp_tree_verify: a vocabulary of %ld (at most 2^22)", p->V);
  DSP_REQUIRE(p->max_nodes > 0 && p->max_nodes <= 4096, "dsp_tree_verify: max_nodes=%ld", p->max_nodes);
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
  const size_t smem = (size_t)p->max_nodes * sizeof(int);
  if (p->dtype == DSP_F32)
    DSP_CUDA(launch_plain(tree_verify_kernel<float>, dim3((unsigned)p->S), dim3(THREADS), smem, stream, a));
  else
    DSP_CUDA(launch_plain(tree_verify_kernel<bf16>, dim3((unsigned)p->S), dim3(THREADS), smem, stream, a));
  DSP_CHECK_LAUNCH("dsp_tree_verify");
  return 0;
}
