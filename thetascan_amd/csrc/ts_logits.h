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

// 2^(j / 64)
static __device__ const double kPowers64[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

// e^t for t in [-745, 0], to some 2^-52 of itself, by a table and a short polynomial (the table-driven
// method of P. T. P. Tang, 1989): t = n ln 2 / 64 + r, 2^(n / 64) from the table above (or a copy in
// LDS), e^r by its series.
struct Exp64 {
  const double* table;
  __device__ __forceinline__ double operator()(double t) const {
    const double k = rint(t * (64.0 / kLn2));
    const int n = (int)k;
    double r = fma(k, -0x1.62e42fefap-7, t);  // ln 2 / 64 in two parts
    r = fma(k, -0x1.cf79abc9e3b3ap-46, r);
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    return __builtin_ldexp(e * table[n & 63], n >> 6);
  }
  // round(2^44 e^t) for t in [-32, 0]: the whole parts come from the low bits of sums with 3 2^51 and 2^52, and
  // the powers of two go into the exponent's bits (conversions and scalings take four times as long).
  __device__ __forceinline__ unsigned long long whole(double t) const {
    const double m = fma(t, 64.0 / kLn2, 0x1.8p52), k = m - 0x1.8p52;
    const int n = (int)(uint32_t)__double_as_longlong(m);
    double r = fma(k, -0x1.62e42fefap-7, t);
    r = fma(k, -0x1.cf79abc9e3b3ap-46, r);
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    const long long scaled = __double_as_longlong(e * table[n & 63]) + ((long long)((n >> 6) + 44) << 52);
    return (unsigned long long)(__double_as_longlong(__longlong_as_double(scaled) + 0x1p52) - __double_as_longlong(0x1p52));
  }
};

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
