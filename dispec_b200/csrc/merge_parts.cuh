// Joins partial results of a row: part k has a largest score m_k (base-2 domain), l_k = sum 2^(s - m_k) and four columns of
// a_k = sum 2^(s - m_k) v; the result is sum a_k 2^(m_k - M) / sum l_k 2^(m_k - M), M = max m_k, 0 where there is no key.
// `load(k, ml, a)` brings part k.  Parts are asked for so many at a time, maxima, sums and outputs together.
#pragma once
#include "common.cuh"

struct Merged {
  float4 sum;        // of weights times values, four columns
  float top, total;  // the largest score (base-2 domain) and the sum of weights, both relative to it
};
template <int AT_ONCE = 8, typename Load>
__device__ __forceinline__ Merged merge_parts(int parts, Load load) {
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < parts; k0 += AT_ONCE) {
    float4 v[AT_ONCE];
    float2 p[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) load(min(k0 + k, parts - 1), p[k], v[k]);
    float top = M;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      if (k0 + k >= parts) p[k] = make_float2(-INFINITY, 0.f);
      top = fmaxf(top, p[k].x);
      // a part without a largest score saw no key, and its sum is 0; or scores that are no numbers, and neither is its sum
      if (p[k].x == -INFINITY) L += p[k].y;
    }
    if (top == -INFINITY) continue;
    const float w0 = exp2f(M - top);
    L *= w0;
    acc = make_float4(acc.x * w0, acc.y * w0, acc.z * w0, acc.w * w0);
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      if (p[k].x == -INFINITY) continue;
      const float w = exp2f(p[k].x - top);
      L = fmaf(w, p[k].y, L);
      acc = make_float4(fmaf(w, v[k].x, acc.x), fmaf(w, v[k].y, acc.y), fmaf(w, v[k].z, acc.z), fmaf(w, v[k].w, acc.w));
    }
    M = top;
  }
  return {acc, M, L};
}
__device__ __forceinline__ float4 merged(const Merged& x) {
  const float inv = x.total == 0.f ? 0.f : 1.f / x.total;  // (NaN stays)
  return make_float4(x.sum.x * inv, x.sum.y * inv, x.sum.z * inv, x.sum.w * inv);
}
