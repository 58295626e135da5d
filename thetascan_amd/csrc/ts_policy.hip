// Clipped policy loss with a KL term on (soft-capped) logits, forward and
// backward (gfx950).
//
//   y = cap tanh(z / cap) (or z);  lp = y_tok - log sum_v e^{y_v};  r = e^{lp - old}
//   loss = sum_n w_n [ -min(r A, clip(r, 1 - low, 1 + high) A) + kl (e^{ref - lp} - (ref - lp) - 1) ]
//   dloss/dlp = w [ -r A where not clipped + kl (1 - e^{ref - lp}) ]
//   dz_v = dloss/dlp (1[v = tok] - e^{y_v - lse}) (1 - (y_v / cap)^2)
//
// Bound by the logits' bytes (65536 rows of 1024 bf16, capped: gradient 53 us at 5.1 TB/s; its
// scan by its arithmetic, 57 us for 134 MB; 8192 rows of 32768: both 239 us, 4.5 TB/s of what
// has to move): a row is
// scanned by one wave (or by a workgroup where it is long) with a running maximum and
// sum, and its gradient is formed by the same workgroup right after (long rows in
// training) or by a kernel of its own; few long rows are scanned by several workgroups
// each.  The sums of exponentials are fp32; a row's own terms are formed in fp64, for
// several rows at once (a lane each, after the rows of its wave), and the rows are
// added in fp64 in a fixed order: normalized advantages all but cancel in the sum.  A
// row of weight zero is not read; its log-probability is given as zero, its gradient
// too.

#include "ts_common.h"
#include "ts_tokens.h"

#include <string.h>

namespace ts {

constexpr float kLog2eF = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;
struct PolicyP {
  int64_t rows, stride;
  int V;
  float cap;
  double kl, low, high;
  const void* z;
  const int64_t* tokens;
  const float *old, *ref, *adv, *w;
  float *lp, *coef;
  float* lse;  // [2][rows]: the maximum, and log2 of the sum of e^{x - maximum}
  double* part;
  float2* scans;  // [rows][split], where split is not one
  int split;
  const float* g;
  void* dz;
  int formed;  // dz holds the gradient for g = 1: nothing is left to do there
};

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

// One row's terms from its maximum and sum, in fp64.  Where the token is the maximum, its
// distance from it is zero: the capped maximum is rounded to fp32, and a difference from the
// token's exact value would give log-probabilities above zero.
template <typename E, bool CAP>
__device__ __forceinline__ void row_terms(const PolicyP& p, int64_t n, float w, float m, float s, float& lpf, float& coef,
                                          float& logs, double& term) {
  const double l2 = log2((double)s);
  const int64_t tok = p.tokens[n];
  double off = (double)NAN;  // the token's logit from the maximum; of a token that is none of the row's
  if (tok >= 0 && tok < p.V) {
    const float z = tof(((const E*)p.z)[n * p.stride + tok]);
    double y = (double)z;
    if (CAP) y = (double)p.cap * tanh(y / (double)p.cap);
    off = CAP && Logit<CAP>(p.cap).any(z) >= m ? 0.0 : y - (double)m;
  }
  const double lp = off - l2 * kLn2;
  logs = (float)l2;
  lpf = (float)lp;
  if (!p.adv) return;
  const double A = (double)p.adv[n], r = exp(lp - (double)p.old[n]);
  const double edge = A > 0.0 ? 1.0 + p.high : 1.0 - p.low;
  const bool flat = (A > 0.0 && r > edge) || (A < 0.0 && r < edge);
  term = -(flat ? edge : r) * A;
  double slope = flat ? 0.0 : -r * A;
  if (p.ref) {
    const double d = (double)p.ref[n] - lp, e = expm1(d);
    term += p.kl * (e - d);
    slope -= p.kl * e;
  }
  term *= (double)w;
  coef = (float)(slope * (double)w);
}

constexpr int kScan = 4;  // vectors a thread has on their way at once
// This thread's share (of LANES) of a row's running maximum and sum: part `part` of
// `parts` of its vectors, and its ends with the first.
template <typename E, bool CAP, int LANES>
__device__ __forceinline__ void row_scan(const E* row, int V, const Logit<CAP>& f, int li, float& m, float& s,
                                         int part = 0, int parts = 1) {
  constexpr int N = Vec16<E>::N, U = kScan;
  const RowSpan<E> span(row, V);
  const Vec16<E>* vec = (const Vec16<E>*)(row + span.head);
  m = kLowest;
  s = 0.f;
  auto one = [&](float x) {
    const float top = fmaxf(m, x);
    s = fmaf(s, ex(m - top), ex(x - top));
    m = top;
  };
  for (int i = li + part * LANES * U; i < span.vecs; i += parts * LANES * U) {
    Vec16<E> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * LANES < span.vecs) v[u].raw = vec[i + u * LANES].raw;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * LANES < span.vecs) {
        float x[N], top = m;
        if (f.some_far(v[u])) {
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = f.any(tof(v[u].e[j]));
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = f.near(tof(v[u].e[j]));
        }
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, x[j]);
        s *= ex(m - top);
#pragma unroll
        for (int j = 0; j < N; ++j) s += ex(x[j] - top);
        m = top;
      }
  }
  if (part == 0) {
    if (li < span.head) one(f.any(tof(row[li])));
    for (int i = span.head + span.vecs * N + li; i < V; i += LANES) one(f.any(tof(row[i])));
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64), top = fmaxf(m, m2);
    s = s * ex(m - top) + s2 * ex(m2 - top);
    m = top;
  }
}

// This thread's share of a row's gradient c dlp/dz: parts of the row's vectors
// (part of parts), and its ends with the first part.
template <typename E, bool CAP, int LANES>
__device__ __forceinline__ void row_grad(const E* row, E* out, int V, bool read, const Logit<CAP>& f, float c, float top,
                                         float logs, int64_t tok, int li, int part, int parts) {
  constexpr int N = Vec16<E>::N, U = 4;
  auto part_of = [&](float x, float slope, int v) {
    const float prob = __builtin_amdgcn_exp2f(fmaf(x - top, kLog2eF, -logs));
    return c * ((v == tok ? 1.f : 0.f) - prob) * slope;
  };
  auto grad = [&](float z, int v) {
    float x;
    const float slope = f.slope_any(z, x);
    return part_of(x, slope, v);
  };
  auto grad_near = [&](float z, int v) {
    const float x = f.near(z);
    return part_of(x, f.slope_near(x), v);
  };
  // the output's vectors; where the logits' do not start with them, they are read element by element
  const RowSpan<E> span(out, V);
  const bool together = (((uintptr_t)(row + span.head)) & 15) == 0;
  for (int i = li + part * LANES * U; i < span.vecs; i += parts * LANES * U) {
    Vec16<E> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].raw = make_uint4(0u, 0u, 0u, 0u);
      const int at = i + u * LANES;
      if (at < span.vecs && read) {
        if (together)
          v[u].raw = ((const Vec16<E>*)(row + span.head))[at].raw;
        else
#pragma unroll
          for (int j = 0; j < N; ++j) v[u].e[j] = row[span.head + at * N + j];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i + u * LANES;
      if (at < span.vecs) {
        Vec16<E> o;
        o.raw = make_uint4(0u, 0u, 0u, 0u);
        if (read && f.some_far(v[u])) {
#pragma unroll
          for (int j = 0; j < N; ++j) o.e[j] = cvt<E>(grad(tof(v[u].e[j]), span.head + at * N + j));
        } else if (read) {
#pragma unroll
          for (int j = 0; j < N; ++j) o.e[j] = cvt<E>(grad_near(tof(v[u].e[j]), span.head + at * N + j));
        }
        ((Vec16<E>*)(out + span.head))[at].raw = o.raw;
      }
    }
  }
  if (part) return;
  if (li < span.head) out[li] = read ? cvt<E>(grad(tof(row[li]), li)) : (E)0.0f;
  for (int i = span.head + span.vecs * N + li; i < V; i += LANES) out[i] = read ? cvt<E>(grad(tof(row[i]), i)) : (E)0.0f;
}

// WPR waves a row, R rows one after the other whose terms are formed together.
template <typename E, bool CAP, int WPR, int R>
__global__ __launch_bounds__(256) void policy_fwd_kernel(PolicyP p) {
  constexpr int THREADS = 256, GROUPS = THREADS / (64 * WPR), LANES = 64 * WPR;
  __shared__ float sm[WPR == 1 ? 1 : THREADS / 64], ss[WPR == 1 ? 1 : THREADS / 64];
  __shared__ double sums[THREADS / 64];
  const int tid = threadIdx.x, lane = tid & 63, gi = tid / LANES, li = tid % LANES;
  const int64_t row0 = ((int64_t)blockIdx.x * GROUPS + gi) * R;
  const Logit<CAP> f(p.cap);
  float mine_m = 0.f, mine_s = 1.f;  // of the row this lane finishes
  for (int k = 0; k < R; ++k) {
    const int64_t n = row0 + k;
    // (uniform over the row's threads; with several waves a row over the workgroup)
    if (n >= p.rows) break;
    if (p.w && p.w[n] == 0.f) continue;
    const E* row = (const E*)p.z + n * p.stride;
    float m, s;
    row_scan<E, CAP, LANES>(row, p.V, f, li, m, s);
    if constexpr (WPR > 1) {
      const int w0 = gi * WPR;
      if (lane == 0) {
        sm[tid >> 6] = m;
        ss[tid >> 6] = s;
      }
      __syncthreads();
      m = kLowest;
#pragma unroll
      for (int w = 0; w < WPR; ++w) m = fmaxf(m, sm[w0 + w]);
      s = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) s = fmaf(ss[w0 + w], ex(sm[w0 + w] - m), s);
      __syncthreads();
    }
    if (li == k) {
      mine_m = m;
      mine_s = s;
    }
  }
  // the rows' own terms, a lane each
  double term = 0.0;
  const int64_t n = row0 + li;
  if (li < R && n < p.rows) {
    const float w = p.w ? p.w[n] : 1.f / (float)p.rows;
    float coef = 0.f, logs = 0.f, lpf = 0.f;
    if (w != 0.f) row_terms<E, CAP>(p, n, w, mine_m, mine_s, lpf, coef, logs, term);
    p.lp[n] = lpf;
    if (p.coef) {
      p.coef[n] = coef;
      p.lse[n] = mine_m;
      p.lse[p.rows + n] = logs;
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int o = R / 2; o >= 1; o >>= 1) term += __shfl_xor(term, o, 64);
  if (lane == 0) sums[tid >> 6] = term;
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int i = 0; i < GROUPS; ++i) total += sums[i * WPR];
    p.part[blockIdx.x] = total;
  }
}

// Few long rows: a row's scan in `split` workgroups, each leaving its maximum and sum,
template <typename E, bool CAP>
__global__ __launch_bounds__(256) void policy_scan_kernel(PolicyP p) {
  __shared__ float sm[4], ss[4];
  const int tid = threadIdx.x;
  const int64_t n = blockIdx.x;
  if (p.w && p.w[n] == 0.f) return;  // uniform
  float m, s;
  row_scan<E, CAP, 256>((const E*)p.z + n * p.stride, p.V, Logit<CAP>(p.cap), tid, m, s, (int)blockIdx.y, p.split);
  if ((tid & 63) == 0) {
    sm[tid >> 6] = m;
    ss[tid >> 6] = s;
  }
  __syncthreads();
  if (tid) return;
  m = kLowest;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(m, sm[i]);
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(ss[i], ex(sm[i] - m), s);
  p.scans[n * p.split + blockIdx.y] = make_float2(m, s);
}
// and the rows' own terms from those, a lane each.
template <typename E, bool CAP>
__global__ __launch_bounds__(64) void policy_join_kernel(PolicyP p) {
  const int64_t n = (int64_t)blockIdx.x * 64 + threadIdx.x;
  double term = 0.0;
  if (n < p.rows) {
    const float w = p.w ? p.w[n] : 1.f / (float)p.rows;
    float coef = 0.f, logs = 0.f, lpf = 0.f, m = 0.f, s = 0.f;
    if (w != 0.f) {
      m = kLowest;
      for (int i = 0; i < p.split; ++i) m = fmaxf(m, p.scans[n * p.split + i].x);
      for (int i = 0; i < p.split; ++i) {
        const float2 one = p.scans[n * p.split + i];
        s = fmaf(one.y, ex(one.x - m), s);
      }
      row_terms<E, CAP>(p, n, w, m, s, lpf, coef, logs, term);
    }
    p.lp[n] = lpf;
    if (p.coef) {
      p.coef[n] = coef;
      p.lse[n] = m;
      p.lse[p.rows + n] = logs;
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) term += __shfl_xor(term, o, 64);
  if (threadIdx.x == 0) p.part[blockIdx.x] = term;
}

// The sum of the workgroups' parts, in a fixed order.
__global__ __launch_bounds__(1024) void policy_sum_kernel(const double* part, int64_t n, float* loss) {
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

template <typename E, bool CAP, int WPR>
__global__ __launch_bounds__(256) void policy_bwd_kernel(PolicyP p) {
  constexpr int LANES = 64 * WPR, GROUPS = 256 / LANES;
  const int tid = threadIdx.x, gi = tid / LANES, li = tid % LANES;
  const int64_t n = (int64_t)blockIdx.x * GROUPS + gi;
  if (n >= p.rows || (p.formed && p.g[0] == 1.f)) return;
  const float c = p.coef[n] * p.g[0], top = p.lse[n], logs = p.lse[p.rows + n];
  const int64_t tok = p.tokens[n];
  const bool read = !p.w || p.w[n] != 0.f;
  row_grad<E, CAP, LANES>((const E*)p.z + n * p.stride, (E*)p.dz + n * (int64_t)p.V, p.V, read, Logit<CAP>(p.cap), c, top,
                          logs, tok, li, (int)blockIdx.y, (int)gridDim.y);
}

// Long rows in training: a workgroup scans a row and forms its gradient (for an
// upstream gradient of one) at once, so that the second reading finds the row in
// the caches: 8192 rows of 32768 bf16 logits 236 us, against 118 and 169 of the two kernels.
template <typename E, bool CAP>
__global__ __launch_bounds__(256) void policy_fused_kernel(PolicyP p) {
  __shared__ float sm[4], ss[4], sc[3];
  const int tid = threadIdx.x;
  const int64_t n = blockIdx.x;
  const float w = p.w ? p.w[n] : 1.f / (float)p.rows;
  const bool read = w != 0.f;  // uniform
  const Logit<CAP> f(p.cap);
  const E* row = (const E*)p.z + n * p.stride;
  float m = 0.f, s = 1.f;
  if (read) {
    row_scan<E, CAP, 256>(row, p.V, f, tid, m, s);
    if ((tid & 63) == 0) {
      sm[tid >> 6] = m;
      ss[tid >> 6] = s;
    }
    __syncthreads();
    m = kLowest;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, sm[i]);
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fmaf(ss[i], ex(sm[i] - m), s);
  }
  if (tid == 0) {
    double term = 0.0;
    float coef = 0.f, logs = 0.f, lpf = 0.f;
    if (read) row_terms<E, CAP>(p, n, w, m, s, lpf, coef, logs, term);
    p.lp[n] = lpf;
    p.coef[n] = coef;
    p.lse[n] = m;
    p.lse[p.rows + n] = logs;
    p.part[n] = term;
    sc[0] = coef;
    sc[1] = logs;
  }
  __syncthreads();
  row_grad<E, CAP, 256>(row, (E*)p.dz + n * (int64_t)p.V, p.V, read, f, sc[0], m, sc[1], p.tokens[n], tid, 0, 1);
}

}  // namespace ts

namespace {

using ts::fail;
using ts::PolicyP;

// Rows of up to 2048 logits take a wave each (no barrier), longer ones a workgroup of
// four.  Forward, bf16: 65536 rows of 1024 51 us with a wave a row, 96 with four; 32768 of
// 2048 46 and 66; 64 of 4096 10 and 7.
int waves_of(const PolicyP& p) { return p.V <= 2048 ? 1 : 4; }

// Workgroups of a row's scan where rows are few and long: each a turn of its loop or
// more (8192 bf16 logits), 1024 in all at most, four at least.  Log-probabilities of 16
// rows of 131072 bf16 logits 8.7 us against 22.8 with a workgroup a row, loss and gradient
// 16.0 against 60.9; 128 rows of 32768 8.2 and 8.7, 17.9 and 22.8; 256 of 32768 10.4 and 9.1,
// 23.9 and 24.8.
int split_of(const PolicyP& p, bool bf) {
  const int64_t turn = 256 * ts::kScan * (bf ? 8 : 4);
  const int64_t fit = p.rows ? 1024 / p.rows : 1, n = p.V / turn;
  const int64_t split = fit < n ? fit : n;
  return split < 4 ? 1 : (int)split;
}

// Whether training forms loss and gradient in one kernel: rows of a workgroup each.
// (Of a wave's rows the fp64 terms are shared, and 65536 rows of 1024 fit the last
// cache between two kernels: one kernel that held them in registers took 113 us
// against 99.)
bool one_pass(const PolicyP& p) { return waves_of(p) == 4 && p.split == 1; }

// A row's fp64 terms cost a wave about as much as 1500 of its logits: where there are
// rows enough to keep every CU busy all the same, eight rows of a wave share one pass
// (forward, rows of 1024: 8192 rows 15.4 us, shared 18.1; 16384 25.2 and 21.5; 65536 79
// and 52).  Rows of a workgroup do not (8192 of 32768: 133 us, shared 155).
bool shares_terms(const PolicyP& p) { return waves_of(p) == 1 && p.rows >= 16384; }

int64_t forward_blocks(const PolicyP& p) {
  if (p.split > 1) return (p.rows + 63) / 64;
  const int64_t per = (waves_of(p) == 1 ? 4 : 1) * (shares_terms(p) ? 8 : 1);
  return (p.rows + per - 1) / per;
}

template <typename E, bool CAP>
void forward(const PolicyP& p, hipStream_t stream) {
  const dim3 grid((unsigned)forward_blocks(p));
  if (p.dz)
    hipLaunchKernelGGL((ts::policy_fused_kernel<E, CAP>), dim3((unsigned)p.rows), dim3(256), 0, stream, p);
  else if (p.split > 1) {
    hipLaunchKernelGGL((ts::policy_scan_kernel<E, CAP>), dim3((unsigned)p.rows, (unsigned)p.split), dim3(256), 0,
                       stream, p);
    hipLaunchKernelGGL((ts::policy_join_kernel<E, CAP>), grid, dim3(64), 0, stream, p);
  } else if (shares_terms(p))
    hipLaunchKernelGGL((ts::policy_fwd_kernel<E, CAP, 1, 8>), grid, dim3(256), 0, stream, p);
  else if (waves_of(p) == 1)
    hipLaunchKernelGGL((ts::policy_fwd_kernel<E, CAP, 1, 1>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((ts::policy_fwd_kernel<E, CAP, 4, 1>), grid, dim3(256), 0, stream, p);
}
template <typename E, bool CAP>
void backward(const PolicyP& p, hipStream_t stream) {
  // a long row's vectors over several workgroups where the rows are few (16 rows of 131072:
  // 5.5 us against 37, 128 of 32768: 7.1 and 12.3)
  const int64_t rows = p.V <= 2048 ? (p.rows + 3) / 4 : p.rows;
  int parts = 1;
  if (p.V > 2048)
    while (rows * parts < 1024 && parts * 8192 < p.V) parts *= 2;
  const dim3 grid((unsigned)rows, (unsigned)parts);
  if (p.V <= 2048)
    hipLaunchKernelGGL((ts::policy_bwd_kernel<E, CAP, 1>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((ts::policy_bwd_kernel<E, CAP, 4>), grid, dim3(256), 0, stream, p);
}

template <typename E>
void forward(const PolicyP& p, hipStream_t stream) {
  return p.cap == 0.f ? forward<E, false>(p, stream) : forward<E, true>(p, stream);
}
template <typename E>
void backward(const PolicyP& p, hipStream_t stream) {
  return p.cap == 0.f ? backward<E, false>(p, stream) : backward<E, true>(p, stream);
}

int setup(const ts_policy_desc* d, const void* z, const int64_t* tokens, PolicyP* p) {
  if (!d || d->rows < 0 || d->V < 1 || d->stride < 0 ||
      !(d->cap == 0.f || (d->cap >= 1e-30f && d->cap <= 1e30f)) || !(d->low >= 0.0 && d->low <= 1.0) ||
      !(d->high >= 0.0) || !(d->kl >= 0.0))
    return fail(TS_ERR_VALUE, "policy_loss: bad shape, cap, clip range or KL coefficient");
  if (d->dtype != TS_BF16 && d->dtype != TS_F32) return fail(TS_ERR_NOT_IMPLEMENTED, "policy_loss: bf16 or fp32 only");
  if (d->rows > 0x7fffffff) return fail(TS_ERR_NOT_IMPLEMENTED, "policy_loss: too many rows");
  if (d->rows && (!z || !tokens || ((uintptr_t)z & (d->dtype == TS_BF16 ? 1u : 3u))))
    return fail(TS_ERR_VALUE, "policy_loss: missing or misaligned logits or tokens");
  memset(p, 0, sizeof(*p));
  p->rows = d->rows; p->V = d->V; p->stride = d->stride; p->cap = d->cap;
  p->kl = d->kl; p->low = d->low; p->high = d->high;
  p->z = z; p->tokens = tokens;
  p->split = split_of(*p, d->dtype == TS_BF16);
  // (a launch counts its threads in 32 bits)
  if (d->rows * 64 * waves_of(*p) >= (int64_t)1 << 32)
    return fail(TS_ERR_NOT_IMPLEMENTED, "policy_loss: too many rows");
  return TS_OK;
}

int finish(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "%s: launch failed: %s", what, hipGetErrorString(e));
  return TS_OK;
}

}  // namespace

extern "C" {

int ts_capture_id(hipStream_t stream, uint64_t* id) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long n = 0;
  const hipError_t e = hipStreamGetCaptureInfo(stream, &status, &n);
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "capture id: %s", hipGetErrorString(e));
  if (id) *id = status == hipStreamCaptureStatusNone ? 0 : n;
  return TS_OK;
}

int ts_policy_loss_parts(const ts_policy_desc* d, int64_t* parts) {
  PolicyP p;
  const int rc = setup(d, (const void*)16, (const int64_t*)16, &p);
  if (rc) return rc;
  // (the scans' results stand behind the sums)
  const int64_t n = forward_blocks(p);
  if (parts) *parts = p.split > 1 ? n + p.rows * p.split : (one_pass(p) && p.rows > n ? p.rows : n);
  return TS_OK;
}

int ts_policy_one_pass(const ts_policy_desc* d, int32_t* yes) {
  PolicyP p;
  const int rc = setup(d, (const void*)16, (const int64_t*)16, &p);
  if (rc) return rc;
  if (yes) *yes = one_pass(p);
  return TS_OK;
}

int ts_policy_loss_fwd(const ts_policy_desc* d, const ts_policy_io* io, hipStream_t stream) {
  PolicyP p;
  if (!io) return fail(TS_ERR_VALUE, "policy_loss: missing tensors");
  const int rc = setup(d, io->logits, io->tokens, &p);
  if (rc) return rc;
  if (d->rows && !io->log_probs) return fail(TS_ERR_VALUE, "policy_loss: no place for the log-probabilities");
  if (io->loss && (!io->parts || (d->rows && (!io->old_log_probs || !io->advantages || !io->coef || !io->lse))))
    return fail(TS_ERR_VALUE, "policy_loss: missing tensors");
  p.old = io->old_log_probs; p.ref = io->ref_log_probs; p.adv = io->loss ? io->advantages : nullptr; p.w = io->weights;
  p.lp = io->log_probs; p.coef = io->loss ? io->coef : nullptr; p.lse = io->lse;
  p.part = io->loss ? io->parts : nullptr;
  if (p.split > 1) {
    if (!io->parts) return fail(TS_ERR_VALUE, "policy_loss: missing parts");
    p.scans = (float2*)(io->parts + forward_blocks(p));
  }
  p.dz = io->loss ? io->dlogits : nullptr;
  if ((uintptr_t)p.dz & 15u) return fail(TS_ERR_VALUE, "policy_loss: misaligned gradient");
  if (p.dz && !one_pass(p))
    return fail(TS_ERR_NOT_IMPLEMENTED, "policy_loss: rows of %d take two passes", p.V);
  if (d->rows) {
    if (d->dtype == TS_BF16)
      forward<ts::bf16>(p, stream);
    else
      forward<float>(p, stream);
  }
  if (io->loss)
    hipLaunchKernelGGL(ts::policy_sum_kernel, dim3(1), dim3(1024), 0, stream, (const double*)io->parts,
                       !d->rows ? 0 : (p.dz ? p.rows : forward_blocks(p)), io->loss);
  return finish("policy_loss");
}

static int policy_bwd(const ts_policy_desc* d, const ts_policy_io* io, const float* dloss, void* dlogits, bool formed,
                      hipStream_t stream) {
  PolicyP p;
  if (!io) return fail(TS_ERR_VALUE, "policy_loss bwd: missing tensors");
  const int rc = setup(d, io->logits, io->tokens, &p);
  if (rc) return rc;
  if (d->rows == 0) return TS_OK;
  if (!io->coef || !io->lse || !dloss || !dlogits || ((uintptr_t)dlogits & (d->dtype == TS_BF16 ? 1u : 3u)))
    return fail(TS_ERR_VALUE, "policy_loss bwd: missing or misaligned tensors");
  p.w = io->weights; p.coef = io->coef; p.lse = io->lse; p.g = dloss; p.dz = dlogits; p.formed = formed;
  if (d->dtype == TS_BF16)
    backward<ts::bf16>(p, stream);
  else
    backward<float>(p, stream);
  return finish("policy_loss bwd");
}

int ts_policy_loss_bwd(const ts_policy_desc* d, const ts_policy_io* io, const float* dloss, void* dlogits,
                       hipStream_t stream) {
  return policy_bwd(d, io, dloss, dlogits, false, stream);
}

int ts_policy_loss_scale(const ts_policy_desc* d, const ts_policy_io* io, const float* dloss, hipStream_t stream) {
  return policy_bwd(d, io, dloss, io ? io->dlogits : nullptr, true, stream);
}

}  // extern "C"
