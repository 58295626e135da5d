// Rows of (soft-capped) logits: what the losses and the sampler share (gfx950).
#pragma once

#include "ts_common.h"
#include "ts_tokens.h"

namespace ts {

constexpr float kLog2eF = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;

// A logit as the softmax takes it: itself, or y = cap tanh(z / cap).  near, for |z| < cap / 2: by
// the series of tanh(t) / t to t^14 (its next term 2^-26 of it), one rounding of z and what the
// cap takes off.  any: beyond that cap - 2 cap r of the size, r = 1 / (1 + e^{2 |z| / cap}), off by
// some 2^-23 of itself.  (near costs what the exponential and the reciprocal do; a wave whose
// logits are all near takes it alone.  By r alone, of z instead of its size, capped logits were
// off by cap 2^-23.)
template <bool CAP>
struct Logit {
  float cap, inv, in, half;
  __device__ __forceinline__ explicit Logit(float c) {
    cap = c;
    inv = CAP ? 1.f / c : 0.f;
    in = CAP ? 2.f * kLog2eF / c : 0.f;
    half = 0.5f * c;
  }
  __device__ __forceinline__ float near(float z) const {
    if (!CAP) return z;
    const float t = z * inv, u = t * t;
    float y = -929569.f / 638512875.f;
    y = fmaf(y, u, 21844.f / 6081075.f);
    y = fmaf(y, u, -1382.f / 155925.f);
    y = fmaf(y, u, 62.f / 2835.f);
    y = fmaf(y, u, -17.f / 315.f);
    y = fmaf(y, u, 2.f / 15.f);
    y = fmaf(y, u, -1.f / 3.f);
    return fmaf(z * u, y, z);
  }
  __device__ __forceinline__ float sig(float z) const { return rcp(1.f + __builtin_amdgcn_exp2f(fabsf(z) * in)); }
  __device__ __forceinline__ float far(float z, float r) const { return copysignf(fmaf(-2.f * cap, r, cap), z); }
  __device__ __forceinline__ float any(float z) const {
    return CAP && !(fabsf(z) < half) ? far(z, sig(z)) : near(z);
  }
  // dy/dz, and y
  __device__ __forceinline__ float slope_near(float y) const {
    const float w = y * inv;
    return CAP ? fmaf(-w, w, 1.f) : 1.f;
  }
  __device__ __forceinline__ float slope_any(float z, float& y) const {
    y = near(z);
    float d = slope_near(y);
    if (CAP) {
      const float r = sig(z);
      if (!(fabsf(z) < half)) {
        y = far(z, r);
        d = 4.f * r * (1.f - r);
      }
    }
    return d;
  }
  // Whether a vector of logits has one past near's range in any lane here.
  template <typename V>
  __device__ __forceinline__ bool some_far(const V& v) const {
    if (!CAP) return false;
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < V::N; ++j) most = fmaxf(most, fabsf(tof(v.e[j])));
    return __any(!(most < half));
  }
};
__device__ __forceinline__ float ex(float d) { return __builtin_amdgcn_exp2f(d * kLog2eF); }
constexpr float kLowest = -3.402823466e38f;

// The parts of a row: `head` elements before its first 16-byte boundary, then
// `vecs` vectors, then a tail.
template <typename E>
struct RowSpan {
  int head, vecs;
  __device__ __forceinline__ RowSpan(const E* row, int V) {
    constexpr int N = Vec16<E>::N;
    head = min(V, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(E)));
    vecs = (V - head) / N;
  }
};

// The sum of the workgroups' parts, in a fixed order.
static __global__ __launch_bounds__(1024) void rows_sum_kernel(const double* part, int64_t n, float* loss) {
  __shared__ double s[1024];
  const int tid = threadIdx.x;
  double sum = 0.0;
  for (int64_t i = tid; i < n; i += 8 * 1024) {  // eight loads on their way at once
    double v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i + u * 1024 < n ? part[i + u * 1024] : 0.0;
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += v[u];
  }
  s[tid] = sum;
  __syncthreads();
  for (int o = 512; o >= 1; o >>= 1) {
    if (tid < o) s[tid] += s[tid + o];
    __syncthreads();
  }
  if (tid == 0) loss[0] = (float)s[0];
}

}  // namespace ts
