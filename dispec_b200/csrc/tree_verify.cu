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
// once: every CTA keeps its share of the row in shared memory, and the CTAs exchange the largest logit and the sums of
// masses through each other's shared memory (one cluster barrier each).  The tests of a node's children need R and a few
// numbers that are read while the row arrives; every CTA makes them for itself, with the same result.
//
// What bounds it: for a few trees the latencies of a node in a row (with 151,936 logits on 16 CTAs the row's arrival 1.05 us, the
// largest logit's exchange 0.55, the pass of exponentials 1.4, the sum's exchange 0.7, the tests 0.45; a refusal against draft
// probabilities 3.5), for many the instructions of the exponentials' pass.  8 trees with draft probabilities 32 us, 64 trees
// without 67 us (1.4 TB/s of the rows that are visited).  A refusal against draft probabilities goes through the masses again, with all
// of the node's refusals: c of them at one node take c (c + 1) / 2 passes.
#include <float.h>

#include "tensor_checks.cuh"
#include "tcgen05_common.cuh"  // bounded mbarrier waits, cluster addresses, counted remote stores

namespace {
constexpr int THREADS = 512, WARPS = THREADS / 32, MAX_CTAS = 16, MAX_NODES = 1024;
// Logits of a row that a CTA should have at most, without and with draft probabilities beside them.  Two CTAs fit an SM up to some 23,600
// and 11,300.  With draft probabilities it stays with that (32 trees of 95,000 logits: 67 us on 16 CTAs each, 78 on eight, which
// do not fit twice); without, eight CTAs alone on their SMs are better than 16 in pairs (64 trees of 188,000 logits: 64 and 78 us).
constexpr int SHARE = 24 * 1024, SHARE_DRAFT = 11 * 1024;
constexpr int MAX_VOCAB = 3 << 17;    // 24,576 logits in each of 16 CTAs
typedef long long mass_t;
constexpr mass_t ONE = (mass_t)1 << 40;

struct Args {
  const void* logits;
  const float* draft;
  const int *tokens, *parents, *node_start;
  const float *temperature, *uniforms, *draws;
  int *path, *count, *token;
  long ld, ldq;
  int rows, V, share, max_nodes;
  int* err;
};

__device__ __forceinline__ mass_t warp_sum_mass(mass_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ mass_t mass_of(float e) { return (mass_t)(e * 1099511627776.f); }

// exp(l / temp - top) with the correctly rounded quotient; 0 for a logit that is no number.
//   UNIT     temp is 1
//   PLAIN    inv = 1 / temp rounded once and two of Markstein's corrections q <- q + inv (l - q temp), which round the quotient
//            correctly where nothing over- or underflows (temp and the largest logit are far from that).  A quotient of
//            -inf comes out as no number, whose exponential is 0 as it should be; one so small that a remainder
//            is not exact changes no exponential.  Five instructions for a division's ten, and no reciprocal.
//   GENERAL  a division; the largest logit may be infinite
enum Mode { UNIT, PLAIN, GENERAL };
struct Scale {
  float temp, inv, top;
  Mode mode;
  template <Mode M>
  __device__ __forceinline__ float exponential(float l) const {
    float x = l;
    if (M == PLAIN) {
      float q = l * inv;
      q = fmaf(fmaf(-q, temp, l), inv, q);
      x = fmaf(fmaf(-q, temp, l), inv, q);
    }
    if (M == GENERAL) x = __fdiv_rn(l, temp);
    const float e = fmaxf(expf(x - top), 0.f);
    return M == GENERAL && x == top ? 1.f : e;
  }
  __device__ __forceinline__ float exponential(float l) const {
    return mode == UNIT ? exponential<UNIT>(l) : mode == PLAIN ? exponential<PLAIN>(l) : exponential<GENERAL>(l);
  }
};

__device__ __forceinline__ void near(const void* p, int bytes) {  // into the L2
  for (int i = threadIdx.x * 128; i < bytes; i += THREADS * 128)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p) + i));
}

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(THREADS, 2)
tree_verify_kernel(const Args a) {
  extern __shared__ __align__(16) float xs[];  // [share] this CTA's part of the row; with draft probabilities [share] of them
  __shared__ __align__(8) uint64_t bar[2];     // exchange k uses box and barrier k % 2
  __shared__ __align__(8) float2 box[2][MAX_CTAS];
  __shared__ int parents[MAX_NODES], tokens[MAX_NODES];
  __shared__ float uniforms[MAX_NODES];
  __shared__ float cand_x[MAX_NODES], cand_q[DRAFT ? MAX_NODES : 1];  // logit and draft probability of the present node's children
  __shared__ int gone[DRAFT ? 1 : MAX_NODES];    // refused tokens, without draft probabilities
  __shared__ float left[DRAFT ? MAX_NODES : 1];  // R at each refusal, with them
  __shared__ float warp_value[WARPS];
  __shared__ mass_t warp_mass[WARPS];
  __shared__ mass_t cta_mass[MAX_CTAS];  // the masses of every CTA's part
  __shared__ float sh_top;
  __shared__ mass_t total;  // R
  __shared__ int decided, refused, broken;

  const int ctas = gridDim.y, rank = blockIdx.y;  // (a cluster is the CTAs of one blockIdx.x)
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float* qs = xs + a.share;
  if (tid == 0) {
    for (int k = 0; k < 2; ++k) {
      tc::mbar_init(&bar[k], 1);
      tc::mbar_expect_tx(&bar[k], (uint32_t)ctas * 8u);
    }
    broken = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // every CTA of the cluster is there, its barriers with it, before another one writes to it (waited for below)
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();
  const int first = a.node_start[s], last = a.node_start[s + 1];
  const bool inside = first >= 0 && first <= last && last <= a.rows;
  const int n = inside ? min(last - first, a.max_nodes) : 0;
  if (!inside && rank == 0 && tid == 0) atomicOr(a.err, DSP_ERR_BAD_TREE);  // (as a tree without nodes)
  // (infinite logits share the mass at any temperature, but by an infinite one they could not be divided)
  const float given = a.temperature[s], temp = given > FLT_MAX ? FLT_MAX : given;
  const int begin = min(a.V, rank * a.share), end = min(a.V, begin + a.share), mine = end - begin;
  const int per = ((mine + THREADS - 1) / THREADS) | 1;  // logits of a thread: neighbours, and odd, so that banks do not meet
  if (n > 0) near((const T*)a.logits + (size_t)first * a.ld + begin, mine * (int)sizeof(T));
  int* path = a.path + (size_t)s * a.max_nodes;
  if (rank == 0)
    for (int i = tid; i < a.max_nodes; i += THREADS) path[i] = i == 0 && n > 0 ? 0 : -1;
  for (int i = tid; i < n; i += THREADS) {
    const int t = a.tokens[first + i];
    parents[i] = a.parents[first + i];
    uniforms[i] = a.uniforms[first + i];
    tokens[i] = t >= 0 && t < a.V ? t : -1;
    if (i > 0 && (t < 0 || t >= a.V)) atomicOr(a.err, DSP_ERR_BAD_TOKEN);  // (the root is not tried)
  }
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (n <= 0) {  // (the whole cluster leaves)
    if (rank == 0 && tid == 0) {
      a.count[s] = 0;
      a.token[s] = -1;
    }
    return;
  }

  int turn = 0, phases = 0;  // bit k of `phases`: the parity that barrier k is waited for with
  // By warp 0: sends eight bytes to every CTA of the cluster and returns, in lane r, what CTA r sent.  Nobody writes to a box
  // that is still being read: a box is used again two exchanges later, which takes a message from here in between.
  auto exchange = [&](float2 v) -> float2 {
    if (ctas == 1) return v;
    if (lane < ctas)
      tc::st_async_v2(tc::mapa_u32(tc::smem_u32(&box[turn][rank]), (uint32_t)lane), v,
                      tc::mapa_u32(tc::smem_u32(&bar[turn]), (uint32_t)lane));
    if (!broken && !__all_sync(0xffffffffu, tc::mbar_wait(&bar[turn], (phases >> turn) & 1))) {
      if (lane == 0) {
        broken = 1;  // the numbers are worthless from here on; nothing waits any more
        atomicOr(a.err, DSP_ERR_WAIT_LIMIT);
      }
      __syncwarp();
    }
    if (lane == 0) tc::mbar_expect_tx(&bar[turn], (uint32_t)ctas * 8u);
    const float2 got = box[turn][lane & (MAX_CTAS - 1)];
    phases ^= 1 << turn;
    turn ^= 1;
    __syncwarp();
    return got;
  };
  // the largest of all threads' values in the cluster
  auto cluster_max = [&](float v) -> float {
    v = warp_max(v);
    if (lane == 0) warp_value[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = warp_max(lane < WARPS ? warp_value[lane] : -INFINITY);
      const float2 got = exchange(make_float2(v, 0.f));
      v = warp_max(lane < ctas ? got.x : -INFINITY);
      if (lane == 0) sh_top = v;
    }
    __syncthreads();
    return sh_top;
  };
  // By warp 0, behind a block barrier: the sum of the warps' masses in the cluster, and in lane r that of CTA r.
  auto cluster_sum = [&](mass_t& each) -> mass_t {
    const mass_t v = warp_sum_mass(lane < WARPS ? warp_mass[lane] : 0);
    const float2 got = exchange(make_float2(__int_as_float((int)(v & 0xffffffffll)), __int_as_float((int)(v >> 32))));
    each = lane < ctas ? ((mass_t)__float_as_int(got.y) << 32) | (mass_t)(uint32_t)__float_as_int(got.x) : 0;
    return warp_sum_mass(each);
  };

  int cur = 0, count = 1;
  for (;;) {
    // ---- the row of node cur
    const T* row = (const T*)a.logits + (size_t)(first + cur) * a.ld;
    const T* src = row + begin;
    const float* q = DRAFT ? a.draft + (size_t)(first + cur) * a.ldq : nullptr;
    __syncthreads();  // parents are there; nobody reads the last row any more
    // a thread's first child is asked for here and put down behind the requests for the row
    float my_x = 0.f, my_q = 1.f;
    const int my_child = cur + 1 + tid;
    const bool has_child = my_child < n && parents[my_child] == cur && tokens[my_child] >= 0;
    if (has_child) {
      my_x = to_f32(row[tokens[my_child]]);
      if (DRAFT) my_q = q[tokens[my_child]];
    }
    float top = -INFINITY;
    {
      constexpr int N = 16 / sizeof(T);
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
            for (int c = 0; c < N; c += 4) {
              const float4 x = make_float4(to_f32(l[c]), to_f32(l[c + 1]), to_f32(l[c + 2]), to_f32(l[c + 3]));
              *reinterpret_cast<float4*>(xs + i * N + c) = x;
              top = fmaxf(top, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)));  // (no number is smaller than any)
            }
          }
        }
        done = pieces * N;
      }
#pragma unroll 4
      for (int i = done + tid; i < mine; i += THREADS) {
        const float x = to_f32(src[i]);
        xs[i] = x;
        top = fmaxf(top, x);
      }
    }
    if (has_child) {
      cand_x[my_child] = my_x;
      if (DRAFT) cand_q[my_child] = my_q;
    }
    for (int i = my_child + THREADS; i < n; i += THREADS)
      if (parents[i] == cur && tokens[i] >= 0) {
        cand_x[i] = to_f32(row[tokens[i]]);
        if (DRAFT) cand_q[i] = q[tokens[i]];
      }
    // the node's first child: its row is likely to be read next and comes nearer meanwhile.  A node with children
    // will mostly see one refused, and needs its draft probabilities then.
    int child = 0;
    for (int i0 = cur + 1; i0 < n && child == 0; i0 += 32) {
      const uint32_t is = __ballot_sync(0xffffffffu, i0 + lane < n && parents[min(i0 + lane, n - 1)] == cur);
      if (is != 0u) child = i0 + __ffs(is) - 1;
    }
    if (child != 0) {
      near((const T*)a.logits + (size_t)(first + child) * a.ld + begin, mine * (int)sizeof(T));
      if (DRAFT)
        for (int i = tid; i < mine; i += THREADS)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(qs + i)), "l"(q + begin + i) : "memory");
    }
    top = cluster_max(top);
    const bool alone = !(temp > 0.f) || top == -INFINITY;  // all the mass on the lowest index of `top`
    int first_top = -1;
    Scale scale = {};
    mass_t my_mass = 0;  // of the thread's own logits, per * tid .. per * (tid + 1) - 1
    const int t0 = min(mine, per * tid), t1 = min(mine, t0 + per);
    if (alone) {
      int low = a.V;
      for (int i = tid; i < mine; i += THREADS) {
        const float x = xs[i];
        if (x == top || (top == -INFINITY && isnan(x))) low = min(low, begin + i);  // (no number counts as -inf)
      }
      first_top = (int)-cluster_max((float)-low);  // (whole numbers up to 2^24 are exact)
      const int at = first_top - begin;
      if (at >= t0 && at < t1) my_mass = ONE;
      if (DRAFT)
        for (int i = tid; i < mine; i += THREADS) xs[i] = i == at ? 1.f : 0.f;
      if (tid < ctas) cta_mass[tid] = first_top >= tid * a.share && first_top < (tid + 1) * a.share ? ONE : 0;
      if (tid == 0) total = ONE;
    } else {
      scale.temp = temp;
      scale.inv = __frcp_rn(temp);
      scale.top = __fdiv_rn(top, temp);  // (a quotient grows with its numerator, so this is the largest of them)
      scale.mode = !(fabsf(top) < 1.1e18f && temp > 9.3e-10f && temp < 1.1e9f) ? GENERAL : temp == 1.f ? UNIT : PLAIN;
      auto pass = [&](auto exponential) {
#pragma unroll 4
        for (int i = t0; i < t1; ++i) {
          const float e = exponential(xs[i]);
          if (DRAFT) xs[i] = e;  // refusals come back to them
          my_mass += mass_of(e);
        }
      };
      if (scale.mode == UNIT)
        pass([&](float l) { return scale.exponential<UNIT>(l); });
      else if (scale.mode == PLAIN)
        pass([&](float l) { return scale.exponential<PLAIN>(l); });
      else
        pass([&](float l) { return scale.exponential<GENERAL>(l); });
      const mass_t sum = warp_sum_mass(my_mass);
      if (lane == 0) warp_mass[warp] = sum;
      __syncthreads();
      if (warp == 0) {
        mass_t each;
        const mass_t all = cluster_sum(each);
        if (lane < ctas) cta_mass[lane] = each;
        if (lane == 0) total = all;
        __syncwarp();
      }
    }
    if (tid == 0) refused = 0;
    if (DRAFT) asm volatile("cp.async.wait_all;" ::: "memory");
    if (alone) __syncthreads();  // (else all that follows is warp 0's until the next barrier)

    // ---- its children, in the order of their numbers
    int next = cur + 1;
    for (;;) {
      if (warp == 0) {
        mass_t R = total;
        int found = 0, nr = next == cur + 1 ? 0 : refused;
        for (int i0 = next & ~31; i0 < n && found == 0; i0 += 32) {
          const int me = i0 + lane;
          uint32_t todo = __ballot_sync(0xffffffffu, me >= next && me < n && parents[me] == cur);
          while (todo != 0u && found == 0) {
            const int i = i0 + __ffs(todo) - 1;
            todo &= todo - 1;
            const int t = tokens[i];
            if (t < 0) continue;
            const float u = uniforms[i], e = alone ? (t == first_top ? 1.f : 0.f) : scale.exponential(cand_x[i]);
            mass_t m = mass_of(e);
            if (DRAFT) {
              for (int k = 0; k < nr; ++k) m = max((mass_t)0, m - (mass_t)__fmul_rn(cand_q[i], left[k]));
              if (__fmul_rn(__fmul_rn(u, cand_q[i]), (float)R) < (float)m)
                found = i;
              else
                found = -i;  // refused: the masses have to be summed again
            } else {
              bool was = false;  // refused before: no mass
              for (int k = lane; k < nr; k += 32) was |= gone[k] == t;
              if (__any_sync(0xffffffffu, was)) m = 0;
              if (__fmul_rn(u, (float)R) < (float)m) {
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
          refused = nr;
          if (!DRAFT)
            total = R;
          else if (found < 0)
            left[nr] = (float)R;
        }
      }
      __syncthreads();
      const int decision = decided;
      if (!DRAFT || decision >= 0 || broken) break;
      const int nr = refused + 1;
      mass_t sum = 0;
#pragma unroll 4
      for (int i = t0; i < t1; ++i) {
        mass_t m = mass_of(xs[i]);
        const float qv = qs[i];
        for (int k = 0; k < nr; ++k) m = max((mass_t)0, m - (mass_t)__fmul_rn(qv, left[k]));
        sum += m;
      }
      next = -decision + 1;
      {
        const mass_t of_warp = warp_sum_mass(sum);
        if (lane == 0) warp_mass[warp] = of_warp;
        __syncthreads();
        if (warp == 0) {
          mass_t each;
          const mass_t rest = cluster_sum(each);
          if (rest > 0) {  // (where nothing would be left, the masses stay)
            if (lane < ctas) cta_mass[lane] = each;
            if (lane == 0) {
              total = rest;
              refused = nr;
            }
          }
          __syncwarp();
        }
        __syncthreads();
        if (refused == nr) my_mass = sum;
      }
    }
    const int decision = decided;
    if (decision > 0 && !broken) {
      cur = decision;
      if (rank == 0 && tid == 0) path[count] = cur;
      ++count;
      continue;
    }
    // ---- no child was taken: the draw, by the CTA whose part holds the mass it aims at
    if (broken) {
      // This CTA is ahead of the others, which may still write to its shared memory: it stays until all their threads have given up in
      // their turn (waits are bounded) or are gone, and lets what is on its way land.
      if (rank == 0 && tid == 0) {
        a.count[s] = 0;
        a.token[s] = -1;
      }
      asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;\n\tnanosleep.u32 20000;" ::: "memory");
      return;
    }
    if (rank == 0 && tid == 0) a.count[s] = count;
    const mass_t R = total, aim = max((mass_t)0, min((mass_t)__fmul_rn(a.draws[s], (float)R), R - 1));
    mass_t before = 0;
    for (int r = 0; r < rank; ++r) before += cta_mass[r];
    if (aim < before || aim >= before + cta_mass[rank]) break;
    const int nr = refused;
    auto mass_at = [&](int i) -> mass_t {
      mass_t m = mass_of(DRAFT ? xs[i] : alone ? (begin + i == first_top ? 1.f : 0.f) : scale.exponential(xs[i]));
      if (DRAFT) {
        for (int k = 0; k < nr; ++k) m = max((mass_t)0, m - (mass_t)__fmul_rn(qs[i], left[k]));
      } else {
        for (int k = 0; k < nr; ++k)
          if (gone[k] == begin + i) m = 0;
      }
      return m;
    };
    if (!DRAFT)
      for (int k = 0; k < nr; ++k) {
        const int i = gone[k] - begin;
        if (i >= t0 && i < t1) my_mass -= mass_of(alone ? (gone[k] == first_top ? 1.f : 0.f) : scale.exponential(xs[i]));
      }
    auto scan = [&](mass_t v) -> mass_t {  // inclusive, over a warp
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const mass_t up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
      }
      return v;
    };
    const mass_t upto = scan(my_mass);
    __syncthreads();
    if (lane == 31) warp_mass[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before += warp_mass[w];
    const mass_t mine_from = before + upto - my_mass;
    const uint32_t holds = __ballot_sync(0xffffffffu, mine_from <= aim && aim < mine_from + my_mass);
    if (holds != 0u) {  // one thread of the CTA: its warp looks at its logits, 32 at a time
      const int who = __ffs(holds) - 1, i_end = __shfl_sync(0xffffffffu, t1, who);
      mass_t from = __shfl_sync(0xffffffffu, mine_from, who);
      for (int i0 = __shfl_sync(0xffffffffu, t0, who); i0 < i_end; i0 += 32) {
        const mass_t sums = scan(i0 + lane < i_end ? mass_at(i0 + lane) : 0);
        const uint32_t past = __ballot_sync(0xffffffffu, from + sums > aim);
        if (past != 0u) {
          if (lane == 0) a.token[s] = begin + i0 + __ffs(past) - 1;
          break;
        }
        from += __shfl_sync(0xffffffffu, sums, 31);
      }
    }
    break;
  }
}

template <typename T, bool DRAFT>
int launch(const Args& a, int S, int ctas, cudaStream_t stream) {
  auto kernel = tree_verify_kernel<T, DRAFT>;
  const size_t smem = (size_t)a.share * sizeof(float) * (DRAFT ? 2 : 1);
  static bool allowed[MAX_DEVICES] = {};  // asked for once a device: the largest share, clusters of 16
  const int device = current_device();
  if (device < 0 || !allowed[device]) {
    prefer_max_shared(reinterpret_cast<const void*>(kernel));
    DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  MAX_VOCAB / MAX_CTAS * (int)sizeof(float) * (DRAFT ? 2 : 1)));
    DSP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (device >= 0) allowed[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)S, (unsigned)ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {1, (unsigned)ctas, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  DSP_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return 0;
}
}  // namespace

// tensors: logits, draft probabilities (or none), tokens, parents, node_start, temperature, uniforms, draws, path, count, token.
extern "C" int dsp_tree_verify(const DspTensor* t, const long* options, cudaStream_t stream) {
  const DspTensor &logits = t[0], &draft = t[1], &tokens = t[2], &parents = t[3], &start = t[4], &temperature = t[5], &uniforms = t[6],
                  &draws = t[7], &path = t[8], &count = t[9], &token = t[10];
  const int dev = logits.device;
  const long max_nodes = options[0];
  DSP_REQUIRE(dev >= 0, "verify_tree: CUDA tensors only (there is no CPU path)");
  DSP_REQUIRE(logits.dtype == DSP_T_F32 || logits.dtype == DSP_T_BF16, "verify_tree: kernels exist for float32 and bfloat16 logits");
  DSP_REQUIRE(logits.dims == 2 && logits.stride[1] == 1 && logits.size[1] >= 1 && logits.size[1] <= MAX_VOCAB,
              "verify_tree: logits must be [T, V] with neighbouring columns and V up to %d", MAX_VOCAB);
  DSP_REQUIRE(temperature.dims == 1, "verify_tree: temperature must be one-dimensional");
  const long T = logits.size[0], V = logits.size[1], S = temperature.size[0];
  DSP_REQUIRE(tensor_is(tokens, DSP_T_I32, dev, 1, T) && tensor_is(parents, DSP_T_I32, dev, 1, T) && tensor_is(start, DSP_T_I32, dev, 1, S + 1),
              "verify_tree: tokens [%ld], parents [%ld] and node_start [%ld] must be contiguous int32 on the device of the logits", T, T, S + 1);
  DSP_REQUIRE(tensor_is(temperature, DSP_T_F32, dev, 1, S) && tensor_is(uniforms, DSP_T_F32, dev, 1, T) && tensor_is(draws, DSP_T_F32, dev, 1, S),
              "verify_tree: temperature [%ld], uniforms [%ld] and draws [%ld] must be contiguous float32 on the device of the logits", S, T, S);
  DSP_REQUIRE(draft.dims < 0 || (draft.dtype == DSP_T_F32 && draft.device == dev && draft.dims == 2 && draft.size[0] == T &&
                                 draft.size[1] == V && draft.stride[1] == 1),
              "verify_tree: draft_probs must be float32 [%ld, %ld] with neighbouring columns", T, V);
  DSP_REQUIRE(max_nodes >= 1 && max_nodes <= MAX_NODES, "verify_tree: max_nodes %ld outside 1 .. %d", max_nodes, MAX_NODES);
  DSP_REQUIRE(tensor_is(path, DSP_T_I32, dev, 2, S, max_nodes) && tensor_is(count, DSP_T_I32, dev, 1, S) && tensor_is(token, DSP_T_I32, dev, 1, S),
              "verify_tree: results must be contiguous int32");
  DSP_REQUIRE(T <= 0x7fffffff && S <= 0x7fffffff, "verify_tree: sizes out of range");
  if (S == 0) return 0;
  Args a = {};
  a.logits = logits.data;
  a.draft = draft.dims < 0 ? nullptr : (const float*)draft.data;
  a.tokens = (const int*)tokens.data;
  a.parents = (const int*)parents.data;
  a.node_start = (const int*)start.data;
  a.temperature = (const float*)temperature.data;
  a.uniforms = (const float*)uniforms.data;
  a.draws = (const float*)draws.data;
  a.path = (int*)path.data;
  a.count = (int*)count.data;
  a.token = (int*)token.data;
  a.ld = logits.stride[0];
  a.ldq = draft.dims < 0 ? 0 : draft.stride[0];
  a.rows = (int)T;
  a.V = (int)V;
  a.max_nodes = (int)max_nodes;
  a.err = dsp_device_error_ptr();
  DSP_REQUIRE(a.err != nullptr, "verify_tree: no device error word");
  // CTAs a tree: as many as keep the device's SMs busy with the trees there are, at least 2,048 logits each, and so many that no
  // share is larger than it should be (beyond 16 CTAs of that it is)
  const int sms = dsp_num_sms(), fits = a.draft ? SHARE_DRAFT : SHARE;
  int ctas = 1;
  while (ctas < MAX_CTAS && ((V + ctas - 1) / ctas > fits || (ctas * 2 * 2048 <= V && ctas * 2 * S <= 2 * sms))) ctas *= 2;
  a.share = (int)(((V + ctas - 1) / ctas + 7) / 8 * 8);
  const bool f32 = logits.dtype == DSP_T_F32;
  const int rc = f32 ? (a.draft ? launch<float, true>(a, (int)S, ctas, stream) : launch<float, false>(a, (int)S, ctas, stream))
                     : (a.draft ? launch<bf16, true>(a, (int)S, ctas, stream) : launch<bf16, false>(a, (int)S, ctas, stream));
  if (rc != 0) return rc;
  DSP_CHECK_LAUNCH("verify_tree");
  return 0;
}
