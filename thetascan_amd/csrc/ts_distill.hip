// Distillation from a teacher's top tokens on (soft-capped, tempered) logits, forward and backward
// (gfx950).
//
//   x = cap tanh(z / cap) / temperature;  lq = x - log sum_v e^{x_v}
//   loss = sum_n w_n [ sum_k P_k (lp_k - lq_k) + P_r (log P_r - log Q_r) ]
//   dz_v = w / temperature (1 - (y_v / cap)^2) * { M q_v - P_v          of the teacher's tokens
//                                                  q_v (M - P_r / Q_r)  elsewhere }
// with M = sum P_k + P_r.  Bound by the logits' bytes.
//
// The share of all other tokens, Q_r, is small where teacher and student agree: it is summed over
// those tokens alone (the teacher's are marked in LDS, a bit each), from a maximum of their own, not
// taken from one.  Sums of exponentials are fp32; the K tokens' terms are formed and added in fp64
// (they all but cancel), the rows in fp64 in a fixed order.

#include "ts_common.h"
#include "ts_logits.h"
#include "ts_tokens.h"

#include <string.h>

namespace ts {

struct DistillP {
  int64_t rows, stride;
  int V, K, tail;
  float cap;
  double inv_t;
  const void* z;
  const int64_t* ids;
  const float *lps, *w;
  float *each, *stats;
  double* part;
  const float* g;
  void* dz;
};

// What the backward takes of a row: the others' maximum and the factor of their e^{x - maximum}; log of
// the sum of all e^x; M; the log of the teacher's sum (0 with a tail).
struct DistillRow {
  float top, rest, lse, mass;
};

// The threads of a row (LANES: a wave, or the workgroup).
template <int LANES>
struct RowTeam {
  double* sm;  // LDS, a value a wave, twice
  int li, wave;
  __device__ __forceinline__ void sync() const {
    if (LANES > 64)
      __syncthreads();
    else
      wave_lds_sync();
  }
  template <typename T, typename F>
  __device__ __forceinline__ T reduce(T x, F f) const {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = f(x, (T)__shfl_xor(x, o, 64));
    if (LANES > 64) {
      __syncthreads();
      if ((li & 63) == 0) sm[wave] = (double)x;
      __syncthreads();
      x = (T)sm[0];
#pragma unroll
      for (int w = 1; w < LANES / 64; ++w) x = f(x, (T)sm[w]);
    }
    return x;
  }
  template <typename T>
  __device__ __forceinline__ T sum(T x) const { return reduce(x, [](T a, T b) { return a + b; }); }
  template <typename T>
  __device__ __forceinline__ T most(T x) const { return reduce(x, [](T a, T b) { return a > b ? a : b; }); }
};

template <bool CAP>
__device__ __forceinline__ double distill_logit(const DistillP& p, float z) {
  double y = (double)z;
  if (CAP) y = (double)p.cap * tanh(y / (double)p.cap);
  return y * p.inv_t;
}

// One row by LANES threads: its loss, and what the backward takes of it.
template <typename E, bool CAP, int LANES>
__device__ __forceinline__ double distill_row(const DistillP& p, int64_t n, const RowTeam<LANES>& team, uint32_t* marks,
                                              DistillRow& out) {
  constexpr int N = Vec16<E>::N;
  const int li = team.li, V = p.V, K = p.K;
  const E* row = (const E*)p.z + n * p.stride;
  const int64_t* ids = p.ids + n * K;
  const float* lps = p.lps + n * K;
  const Logit<CAP> f(p.cap);
  const float inv_t = (float)p.inv_t;
  const int shift = (int)(((uintptr_t)row & 15) / sizeof(E)), vecs = (V + shift + N - 1) / N;
  // the teacher's tokens, a bit each (from the 16-byte boundary at or before the row's start)
  team.sync();
  for (int i = li; i < (vecs * N + 31) / 32; i += LANES) marks[i] = 0;
  team.sync();
  bool bad = false;
  for (int k = li; k < K; k += LANES) {
    const int64_t id = ids[k];
    if (id < 0) continue;
    if (id >= V) {
      bad = true;
      continue;
    }
    const uint32_t bit = (uint32_t)(id + shift);
    bad |= atomicOr(&marks[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1u;
  }
  team.sync();
  // the others: running maximum and sum
  const Vec16<E>* vec = (const Vec16<E>*)(row - shift);
  float m = kLowest, s = 0.f;
  for (int j = li; j < vecs; j += LANES) {
    const int i0 = j * N - shift;
    const uint32_t mark = marks[j * N >> 5] >> (j * N & 31);
    Vec16<E> v;
    float x[N], top = m;
    if (i0 >= 0 && i0 + N <= V) {
      v.raw = vec[j].raw;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v.e[e] = (E)0.f;
        if (i0 + e >= 0 && i0 + e < V) v.e[e] = row[i0 + e];
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[e] = f.any(tof(v.e[e])) * inv_t;
      if (mark >> e & 1u || i0 + e < 0 || i0 + e >= V) x[e] = -INFINITY;
      top = fmaxf(top, x[e]);
    }
    s *= ex(m - top);
#pragma unroll
    for (int e = 0; e < N; ++e) s += ex(x[e] - top);
    m = top;
  }
  const float mr = team.most(m);
  const float sr = team.sum(s * ex(m - mr));
  // the teacher's tokens: the highest of all, the sums, then the terms
  double hi = sr > 0.f ? (double)mr : -INFINITY, mass = 0.0;
  for (int k = li; k < K; k += LANES) {
    const int64_t id = ids[k];
    if (id < 0 || id >= V) continue;
    const double x = distill_logit<CAP>(p, tof(row[id]));
    hi = x > hi ? x : hi;
    mass += exp((double)lps[k]);
  }
  hi = team.most(hi);
  mass = team.sum(mass);
  double total = 0.0;
  for (int k = li; k < K; k += LANES) {
    const int64_t id = ids[k];
    if (id >= 0 && id < V) total += exp(distill_logit<CAP>(p, tof(row[id])) - hi);
  }
  const bool others = sr != 0.f;  // (or no number)
  total = team.sum(total) + (others ? (double)sr * exp((double)mr - hi) : 0.0);
  const double lse = hi + log(total), norm = p.tail ? 0.0 : log(mass);
  double term = 0.0;
  for (int k = li; k < K; k += LANES) {
    const int64_t id = ids[k];
    if (id < 0 || id >= V) continue;
    const double lp = (double)lps[k] - norm, P = exp(lp);
    if (P != 0.0) term += P * (lp - (distill_logit<CAP>(p, tof(row[id])) - lse));
  }
  term = team.sum(term);
  double left = 0.0;
  if (p.tail) {
    left = others ? 1.0 - mass : 0.0;
    left = left < 0.0 ? 0.0 : left;
    if (left != 0.0) term += left * (log(left) - ((double)mr + log((double)sr) - lse));
    mass += left;
  } else {
    mass = mass > 0.0 ? 1.0 : mass;
  }
  if (team.sum(bad ? 1 : 0)) term = (double)NAN;
  out.top = mr;
  out.rest = others ? (float)(mass * exp((double)mr - lse) - left / (double)sr) : 0.f;
  if (term != term) out.rest = NAN;
  out.lse = (float)lse;
  out.mass = (float)mass;
  return term;
}

template <typename E, bool CAP, int LANES>
__global__ __launch_bounds__(256) void distill_fwd_kernel(DistillP p) {
  constexpr int GROUPS = 256 / LANES;
  extern __shared__ uint32_t marks[];
  __shared__ double sm[4], sums[4];
  const int tid = threadIdx.x, gi = tid / LANES, li = tid % LANES;
  const int64_t n = (int64_t)blockIdx.x * GROUPS + gi;
  RowTeam<LANES> team{sm, li, tid >> 6};
  double term = 0.0;
  if (n < p.rows) {  // (uniform over the row's threads)
    const float w = p.w ? p.w[n] : 1.f / (float)p.rows;
    DistillRow r{0.f, 0.f, 0.f, 0.f};
    if (w != 0.f) term = distill_row<E, CAP, LANES>(p, n, team, marks + gi * ((p.V + 15) / 32 + 2), r);
    if (li == 0) {
      p.each[n] = (float)term;
      if (p.stats) {
        p.stats[n] = r.top;
        p.stats[p.rows + n] = r.rest;
        p.stats[2 * p.rows + n] = r.lse;
        p.stats[3 * p.rows + n] = r.mass;
      }
    }
    term = w != 0.f ? term * (double)w : 0.0;
  }
  if (li == 0) sums[gi] = term;
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int i = 0; i < GROUPS; ++i) total += sums[i];
    p.part[blockIdx.x] = total;
  }
}

template <typename E, bool CAP, int LANES>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillP p) {
  constexpr int N = Vec16<E>::N, GROUPS = 256 / LANES;
  __shared__ double sm[4];
  const int tid = threadIdx.x, gi = tid / LANES, li = tid % LANES;
  const int64_t n = (int64_t)blockIdx.x * GROUPS + gi;
  if (n >= p.rows) return;  // (a whole wave, or none of the workgroup)
  RowTeam<LANES> team{sm, li, tid >> 6};
  const int V = p.V;
  const E* row = (const E*)p.z + n * p.stride;
  E* out = (E*)p.dz + n * (int64_t)V;
  const float w = p.w ? p.w[n] : 1.f / (float)p.rows;
  const RowSpan<E> span(out, V);
  if (w == 0.f) {
    Vec16<E> zero;
    zero.raw = make_uint4(0u, 0u, 0u, 0u);
    for (int j = li; j < span.vecs; j += LANES) ((Vec16<E>*)(out + span.head))[j].raw = zero.raw;
    if (li < span.head) out[li] = (E)0.f;
    for (int i = span.head + span.vecs * N + li; i < V; i += LANES) out[i] = (E)0.f;
    return;
  }
  const Logit<CAP> f(p.cap);
  const float inv_t = (float)p.inv_t, c = w * p.g[0] * inv_t;
  const float top = p.stats[n], rest = p.stats[p.rows + n], lse = p.stats[2 * p.rows + n], mass = p.stats[3 * p.rows + n];
  auto other = [&](float z) {
    float y;
    const float slope = f.slope_any(z, y);
    return c * rest * ex(fmaf(y, inv_t, -top)) * slope;
  };
  const bool together = (((uintptr_t)(row + span.head)) & 15) == 0;
  for (int j = li; j < span.vecs; j += LANES) {
    Vec16<E> v, o;
    if (together)
      v.raw = ((const Vec16<E>*)(row + span.head))[j].raw;
    else
#pragma unroll
      for (int e = 0; e < N; ++e) v.e[e] = row[span.head + j * N + e];
#pragma unroll
    for (int e = 0; e < N; ++e) o.e[e] = cvt<E>(other(tof(v.e[e])));
    ((Vec16<E>*)(out + span.head))[j].raw = o.raw;
  }
  if (li < span.head) out[li] = cvt<E>(other(tof(row[li])));
  for (int i = span.head + span.vecs * N + li; i < V; i += LANES) out[i] = cvt<E>(other(tof(row[i])));
  // the teacher's tokens over those
  double norm = 0.0;
  if (!p.tail) {
    for (int k = li; k < p.K; k += LANES) {
      const int64_t id = p.ids[n * p.K + k];
      if (id >= 0 && id < V) norm += exp((double)p.lps[n * p.K + k]);
    }
    norm = log(team.sum(norm));
  }
  __threadfence_block();
  team.sync();
  for (int k = li; k < p.K; k += LANES) {
    const int64_t id = p.ids[n * p.K + k];
    if (id < 0 || id >= V) continue;
    float y;
    const float slope = f.slope_any(tof(row[id]), y);
    const double q = exp(distill_logit<CAP>(p, tof(row[id])) - (double)lse), P = exp((double)p.lps[n * p.K + k] - norm);
    const float d = rest != rest ? rest : (float)((double)mass * q - P);
    out[id] = cvt<E>(c * d * slope);
  }
}

}  // namespace ts

namespace {

using ts::DistillP;
using ts::fail;

int setup(const ts_distill_desc* d, const ts_distill_io* io, DistillP* p) {
  if (!d || !io || d->rows < 0 || d->V < 1 || d->K < 1 || d->stride < 0 ||
      !(d->cap == 0.f || (d->cap >= 1e-30f && d->cap <= 1e30f)) || !(d->temperature >= 1e-6 && d->temperature <= 1e6))
    return fail(TS_ERR_VALUE, "distill: bad shape, cap or temperature");
  if (d->dtype != TS_BF16 && d->dtype != TS_F32) return fail(TS_ERR_NOT_IMPLEMENTED, "distill: bf16 or fp32 only");
  if (d->V > 1 << 20) return fail(TS_ERR_NOT_IMPLEMENTED, "distill: at most 2^20 logits a row, got %d", d->V);
  // (a launch counts its threads in 32 bits)
  if (d->rows >= 1 << 24) return fail(TS_ERR_NOT_IMPLEMENTED, "distill: too many rows");
  if (d->rows && (!io->logits || ((uintptr_t)io->logits & (d->dtype == TS_BF16 ? 1u : 3u)) || !io->ids || !io->log_probs))
    return fail(TS_ERR_VALUE, "distill: missing or misaligned tensors");
  memset(p, 0, sizeof(*p));
  p->rows = d->rows; p->stride = d->stride; p->V = d->V; p->K = d->K; p->tail = d->tail; p->cap = d->cap;
  p->inv_t = 1.0 / d->temperature;
  p->z = io->logits; p->ids = io->ids; p->lps = io->log_probs; p->w = io->weights;
  p->each = io->each; p->stats = io->stats; p->part = io->parts;
  return TS_OK;
}

bool by_wave(int V) { return V <= 2048; }
int64_t blocks_of(const DistillP& p) { return by_wave(p.V) ? (p.rows + 3) / 4 : p.rows; }

template <typename E, bool CAP>
int forward(const DistillP& p, hipStream_t stream) {
  const dim3 grid((unsigned)blocks_of(p));
  const int lds = ((p.V + 15) / 32 + 2) * 4 * (by_wave(p.V) ? 4 : 1);
  if (by_wave(p.V)) {
    hipLaunchKernelGGL((ts::distill_fwd_kernel<E, CAP, 64>), grid, dim3(256), lds, stream, p);
  } else {
    const hipError_t e = ts::ensure_lds_limit((const void*)ts::distill_fwd_kernel<E, CAP, 256>, (1 << 17) + 8);
    if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "distill: %s", hipGetErrorString(e));
    hipLaunchKernelGGL((ts::distill_fwd_kernel<E, CAP, 256>), grid, dim3(256), lds, stream, p);
  }
  return TS_OK;
}

template <typename E, bool CAP>
int backward(const DistillP& p, hipStream_t stream) {
  const dim3 grid((unsigned)blocks_of(p));
  if (by_wave(p.V))
    hipLaunchKernelGGL((ts::distill_bwd_kernel<E, CAP, 64>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((ts::distill_bwd_kernel<E, CAP, 256>), grid, dim3(256), 0, stream, p);
  return TS_OK;
}

int finish(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "%s: launch failed: %s", what, hipGetErrorString(e));
  return TS_OK;
}

}  // namespace

extern "C" {

int ts_distill_parts(const ts_distill_desc* d, int64_t* parts) {
  ts_distill_io io;
  memset(&io, 0, sizeof(io));
  io.logits = io.ids = (const int64_t*)16;
  io.log_probs = (const float*)16;
  DistillP p;
  const int rc = setup(d, &io, &p);
  if (rc) return rc;
  if (parts) *parts = blocks_of(p);
  return TS_OK;
}

int ts_distill_fwd(const ts_distill_desc* d, const ts_distill_io* io, hipStream_t stream) {
  DistillP p;
  int rc = setup(d, io, &p);
  if (rc) return rc;
  if (!io->loss || (d->rows && (!io->each || !io->parts))) return fail(TS_ERR_VALUE, "distill: missing tensors");
  if (d->rows) {
    if (d->dtype == TS_BF16)
      rc = d->cap == 0.f ? forward<ts::bf16, false>(p, stream) : forward<ts::bf16, true>(p, stream);
    else
      rc = d->cap == 0.f ? forward<float, false>(p, stream) : forward<float, true>(p, stream);
    if (rc) return rc;
  }
  hipLaunchKernelGGL(ts::rows_sum_kernel, dim3(1), dim3(1024), 0, stream, (const double*)io->parts,
                     d->rows ? blocks_of(p) : 0, io->loss);
  return finish("distill");
}

int ts_distill_bwd(const ts_distill_desc* d, const ts_distill_io* io, const float* dloss, void* dlogits,
                   hipStream_t stream) {
  DistillP p;
  int rc = setup(d, io, &p);
  if (rc || d->rows == 0) return rc;
  if (!io->stats || !dloss || !dlogits || ((uintptr_t)dlogits & (d->dtype == TS_BF16 ? 1u : 3u)))
    return fail(TS_ERR_VALUE, "distill bwd: missing or misaligned tensors");
  p.g = dloss;
  p.dz = dlogits;
  if (d->dtype == TS_BF16)
    rc = d->cap == 0.f ? backward<ts::bf16, false>(p, stream) : backward<ts::bf16, true>(p, stream);
  else
    rc = d->cap == 0.f ? backward<float, false>(p, stream) : backward<float, true>(p, stream);
  return rc ? rc : finish("distill bwd");
}

}  // extern "C"
