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
// taken from one.  Exponentials are fp32; the K tokens' terms are formed and added in fp64 (they all
// but cancel), as are a row's last sums, the rows in fp64 in a fixed order.  65536 rows of 1024
// (capped, K 32, with gradient): 136 us, of which vector instructions issue in 63 %; 8192 of
// 32768: 272 us, 3.9 TB/s of what has to move.

#include "ts_common.h"
#include "ts_logits.h"
#include "ts_tokens.h"

#include <string.h>
#include <type_traits>

namespace ts {

struct DistillP {
  int64_t rows, stride;
  int V, K, tail, aligned;
  float cap;
  double inv_t;
  const void* z;
  const int64_t* ids;
  const float *lps, *w;
  float *each, *stats;
  double* part;
  const float* g;
  void* dz;
  int formed;  // dz holds the gradient for g = 1: nothing is left to do there
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

// e^{d / temperature} of differences of capped logits, by powers of two: log2(e) / temperature in two parts
// (a factor that is off by 2^-25 is another temperature: of a teacher and student that all but agree, the
// loss is small against what that moves their log-probabilities).
struct TemperedExp {
  float hi, lo;
  __device__ __forceinline__ explicit TemperedExp(double inv_t) {
    const double c = inv_t / kLn2;
    hi = (float)c;
    lo = (float)(c - (double)hi);
  }
  __device__ __forceinline__ float operator()(float d) const {
    d = d < kLowest ? kLowest : d;  // (of -inf the parts' products would cancel to no number)
    return __builtin_amdgcn_exp2f(fmaf(d, hi, d * lo));
  }
};

// ------------------------------------------------ rows that fit in registers

// Sums and maxima over a wave: neighbours by data-parallel moves, then halves by row swaps.
template <typename F>
__device__ __forceinline__ float wave_fold(float x, F f) {
  auto mv = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x = f(x, mv(x, std::integral_constant<int, 0xb1>{}));   // lanes 1, 0, 3, 2
  x = f(x, mv(x, std::integral_constant<int, 0x4e>{}));   // lanes 2, 3, 0, 1
  x = f(x, mv(x, std::integral_constant<int, 0x141>{}));  // the other half of eight
  x = f(x, mv(x, std::integral_constant<int, 0x140>{}));  // of sixteen
  LanePair p = xor16_pair(x);
  p = xor32_pair(f(p.a, p.b));
  return f(p.a, p.b);
}
__device__ __forceinline__ float wave_sum(float x) {
  return wave_fold(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_most(float x) {
  return wave_fold(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ double wave_sum(double x) {
  auto mv = [](double v, auto ctrl) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, decltype(ctrl)::value, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), decltype(ctrl)::value, 0xf, 0xf, false);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
  };
  x += mv(x, std::integral_constant<int, 0xb1>{});
  x += mv(x, std::integral_constant<int, 0x4e>{});
  x += mv(x, std::integral_constant<int, 0x141>{});
  x += mv(x, std::integral_constant<int, 0x140>{});
  auto half = [](double v, auto pair) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const LanePair lo = pair(__uint_as_float((uint32_t)b)), hi = pair(__uint_as_float((uint32_t)(b >> 32)));
    auto both = [](float l, float h) {
      return __longlong_as_double((long long)((uint64_t)__float_as_uint(h) << 32 | __float_as_uint(l)));
    };
    return both(lo.a, hi.a) + both(lo.b, hi.b);
  };
  x = half(x, [](float v) { return xor16_pair(v); });
  return half(x, [](float v) { return xor32_pair(v); });
}

// A share, or an exponential of a distance from a maximum; what is no number stays none.
__device__ __forceinline__ double distill_exp(const Exp64& e64, double t) { return t > -700.0 ? e64(t) : t == t ? 0.0 : t; }

// What a row's loss is formed from: x counts from the highest of all, hi.  Teacher and student that are
// near leave of these terms some 1e-3 of themselves or less, so they are fp64: the logarithm of the
// sum is of the very distance dm, and the teacher's tokens' exponentials are of the distances in a.  (With the
// whole sum in fp32, losses of 1.6e-3 were off by 2.8e-5 of themselves.)  What fp32 rounds in sr moves the
// loss by Q_r - P_r times that.
struct DistillTerms {
  double mass, a;   // sum P, sum P (lp - (x - hi))
  double ek;        // sum of the teacher's tokens' e^{x - hi}
  float sr;         // the others' sum from their own maximum,
  double dm;        // and its distance from hi
};
__device__ __forceinline__ double distill_loss_of(const DistillP& p, const DistillTerms& t) {
  const double lt = log(t.sr != 0.f ? t.ek + (double)t.sr * distill_exp(Exp64{kPowers64}, t.dm) : t.ek);
  if (!p.tail) return t.mass > 0.0 ? t.a / t.mass - log(t.mass) + lt : t.a;
  double loss = t.a + t.mass * lt;
  // (the student has no other token, or forbids them all: 1 - mass may be the rounding of what teacher and
  // student both forbid, so it is no share there)
  const double left = t.sr != 0.f ? 1.0 - t.mass : 0.0;
  if (left > 0.0) loss += left * (log(left) - t.dm - log((double)t.sr) + lt);
  return loss + 0.0 * left;  // (a share that is no number)
}

// What a wave has of a row before it begins: its logits (VPT vectors a lane), which of them are none
// of its own, and the teacher's tokens with their log-probabilities.
template <typename E, int VPT, int KS>
struct DistillIn {
  static constexpr int N = Vec16<E>::N, LANES = 64;
  Vec16<E> v[VPT];
  int shift, vecs;
  int id[KS];
  float lp[KS], w;
  __device__ __forceinline__ void load(const DistillP& p, int64_t n, int li) {
    w = 0.f;
    if (n >= p.rows) return;
    w = p.w ? p.w[n] : 1.f / (float)p.rows;
    const E* row = (const E*)p.z + n * p.stride;
    shift = (int)(((uintptr_t)row & 15) / sizeof(E));
    vecs = (p.V + shift + N - 1) / N;
    if (w == 0.f) return;  // (uniform over the row's threads)
#pragma unroll
    for (int r = 0; r < VPT; ++r) {
      const int j = li + r * LANES, i0 = j * N - shift;
      v[r].raw = make_uint4(0u, 0u, 0u, 0u);
      if (i0 >= 0 && i0 + N <= p.V) {
        v[r].raw = *(const uint4*)(row + i0);
      } else if (j < vecs) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (i0 + e >= 0 && i0 + e < p.V) v[r].e[e] = row[i0 + e];
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = li + s * LANES;
      id[s] = -1;
      lp[s] = -INFINITY;
      if (k < p.K) {
        const int64_t x = p.ids[n * p.K + k];
        id[s] = x < 0 ? -1 : x < p.V ? (int)x : p.V;
        lp[s] = p.lps[n * p.K + k];
      }
    }
  }
  // the student's logits of those
  __device__ __forceinline__ void gather(const DistillP& p, int64_t n, float* zk) const {
    if (w == 0.f) return;
    const E* row = (const E*)p.z + n * p.stride;
#pragma unroll
    for (int s = 0; s < KS; ++s) zk[s] = id[s] >= 0 && id[s] < p.V ? tof(row[id[s]]) : -INFINITY;
  }
  // which elements of vector r are none of the row's
  __device__ __forceinline__ uint32_t ends(int r, int li, int V) const {
    const int i0 = (li + r * LANES) * N - shift;
    const uint32_t before = i0 < 0 ? (1u << min(-i0, N)) - 1u : 0u;
    const uint32_t behind = i0 + N > V ? ~((1u << max(V - i0, 0)) - 1u) : 0u;
    return (before | behind) & ((1u << N) - 1u);
  }
};

// The factors of a row's gradient: M, the teacher's sum without a tail (one over it), one over all
// e^{x - hi}, and the others' factor of e^{x - their maximum}; no number where the row's loss is none.
struct DistillFactors {
  float mass, norm, inv, rest;
  __device__ __forceinline__ float of_teacher(double P, float q) const {
    return rest != rest ? rest : fmaf(mass * q, inv, -((float)P * norm));
  }
};
// (down: of the others' maximum, e^{x - hi}.)  The others' factor M e^{..} / total - P_r / sr is one
// difference, mass down sr - left ek over total sr: what cancels there, as the student comes near the
// teacher, is fp64.
__device__ __forceinline__ DistillFactors distill_factors(const DistillP& p, double mass, double a, double sr, double ek,
                                                          double down) {
  DistillFactors k;
  if (sr == 0.0) down = 0.0;
  const double from = down * sr, left = p.tail && sr != 0.0 ? fmax(1.0 - mass, 0.0) : 0.0;
  k.inv = rcp((float)(from + ek));
  k.mass = p.tail ? (float)(mass + left) : (mass > 0.0 ? 1.f : (float)mass);
  k.norm = p.tail ? 1.f : rcp((float)mass);
  k.rest = sr != 0.0 ? (float)(p.tail ? mass * from - left * ek : k.mass * from) * k.inv * rcp((float)sr) : 0.f;
  if (!(a == a)) k.rest = NAN;
  return k;
}

// A wave takes R rows one after the other, each held in registers from its one reading to its
// gradient; the next row is on its way meanwhile.  The rows' logarithms follow, a lane each.
// (Three waves a SIMD where 16 logits a lane and a token leave the registers for it: with 172 of them, two,
// 65536 rows of 1024 took 169 us instead of 136.)
template <typename E, bool CAP, int VPT, int KS, int R, bool GRAD>
__global__ __launch_bounds__(256, VPT * Vec16<E>::N <= 16 && KS == 1 ? 3 : 1) void distill_rows_kernel(DistillP p) {
  constexpr int N = Vec16<E>::N, LANES = 64, GROUPS = 4, WORDS = LANES * VPT * N / 32 + 1;
  __shared__ uint32_t all_marks[GROUPS][WORDS];
  __shared__ double sums[GROUPS];
  const int tid = threadIdx.x, gi = tid / LANES, li = tid % LANES;
  uint32_t* marks = all_marks[gi];
  const int V = p.V;
  const int64_t row0 = ((int64_t)blockIdx.x * GROUPS + gi) * R;
  const Logit<CAP> f(p.cap);
  const float inv_t = (float)p.inv_t;
  const Exp64 e64{kPowers64};
  const TemperedExp te(p.inv_t);
  DistillTerms mine{1.0, 0.0, 1.0, 0.f, 0.0};
  float mine_w = 0.f, mine_rest = 0.f, mine_hi = 0.f, mine_mr = 0.f, mine_inv = 0.f, mine_mass = 0.f;
  DistillIn<E, VPT, KS> in;
  float zn[KS];
  in.load(p, row0, li);
  in.gather(p, row0, zn);
  for (int rr = 0; rr < R; ++rr) {
    const int64_t n = row0 + rr;
    if (n >= p.rows) break;  // (uniform over the row's threads, as all that follows)
    const float w = in.w;
    const int shift = in.shift, vecs = in.vecs;
    E* out = GRAD ? (E*)p.dz + n * (int64_t)V : nullptr;
    const bool together = GRAD && (((uintptr_t)(out - shift)) & 15) == 0;
    auto put = [&](int j, const Vec16<E>& x) {
      const int i0 = j * N - shift;
      if (together && i0 >= 0 && i0 + N <= V) {
        *(uint4*)(out + i0) = x.raw;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (i0 + e >= 0 && i0 + e < V) out[i0 + e] = x.e[e];
      }
    };
    if (w == 0.f) {
      if (GRAD) {
        Vec16<E> zero;
        zero.raw = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int r = 0; r < VPT; ++r)
          if (li + r * LANES < vecs) put(li + r * LANES, zero);
      }
      if (rr + 1 < R) {
        in.load(p, n + 1, li);
        if (n + 1 < p.rows) in.gather(p, n + 1, zn);
      }
      continue;
    }
    Vec16<E> v[VPT];
    uint32_t ends[VPT];
    int id[KS];
    float lp[KS], zk[KS];
    bool bad = false;
#pragma unroll
    for (int r = 0; r < VPT; ++r) {
      v[r].raw = in.v[r].raw;
      ends[r] = in.ends(r, li, V);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      lp[s] = in.lp[s];
      zk[s] = zn[s];
      bad |= in.id[s] >= V;
      id[s] = in.id[s] < V ? in.id[s] : -1;
    }
    if (rr + 1 < R) in.load(p, n + 1, li);
    for (int i = li; i < WORDS; i += LANES) marks[i] = 0;
    wave_lds_sync();
#pragma unroll
    for (int s = 0; s < KS; ++s)
      if (id[s] >= 0) {
        const uint32_t bit = (uint32_t)(id[s] + shift);
        bad |= atomicOr(&marks[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1u;
      }
    wave_lds_sync();
    // the capped logits and their slopes, the highest, and the sum of all
    float y[VPT][N], sl[VPT][N], yk[KS], slk[KS], hz = -INFINITY, hl = 0.f;
#pragma unroll
    for (int r = 0; r < VPT; ++r) {
      if (f.some_far(v[r])) {
#pragma unroll
        for (int e = 0; e < N; ++e) sl[r][e] = f.slope_any(tof(v[r].e[e]), y[r][e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          y[r][e] = f.near(tof(v[r].e[e]));
          sl[r][e] = f.slope_near(y[r][e]);
        }
      }
      if (ends[r]) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (ends[r] >> e & 1u) y[r][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) hz = fmaxf(hz, y[r][e]);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) slk[s] = f.slope_any(zk[s], yk[s]);
    if (!p.tail) {  // (uniform) shares of the named tokens alone, from the highest
      hl = -INFINITY;
#pragma unroll
      for (int s = 0; s < KS; ++s) hl = id[s] >= 0 ? fmaxf(hl, lp[s]) : hl;
      hl = wave_most(hl);
    }
    const float high = wave_most(hz);
    double all = 0.0;
#pragma unroll
    for (int r = 0; r < VPT; ++r)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x = te(y[r][e] - high);
        all += (double)x;
        sl[r][e] = CAP ? x * sl[r][e] : x;
      }
    double mass = 0.0, a = 0.0, ek = 0.0, near = 0.0, P[KS];
    float q[KS];
    if (KS == 1 && p.K <= 32) {
      // (uniform) the upper lanes have no token: they form the lower ones' e^off while those form P
      const bool on = id[0] >= 0;
      const double off = on ? ((double)yk[0] - (double)high) * p.inv_t : -INFINITY;
      const double lps = on ? (double)lp[0] - (double)hl : -INFINITY;
      const uint64_t bits = (uint64_t)__double_as_longlong(off);
      const LanePair lo = xor32_pair(__uint_as_float((uint32_t)bits)), hi = xor32_pair(__uint_as_float((uint32_t)(bits >> 32)));
      const double up = __longlong_as_double((long long)((uint64_t)__float_as_uint(hi.a) << 32 | __float_as_uint(lo.a)));
      const double x = distill_exp(e64, li < 32 ? lps : up);
      P[0] = li < 32 ? x : 0.0;
      ek = li < 32 ? 0.0 : x;
      q[0] = on ? te(yk[0] - high) : 0.f;
      near = (double)q[0];
      mass = P[0];
      if (P[0] != 0.0) a = P[0] * (lps - off);
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        P[s] = 0.0;
        q[s] = 0.f;
        if (id[s] >= 0) {
          const double off = ((double)yk[s] - (double)high) * p.inv_t, lps = (double)lp[s] - (double)hl;
          // (in fp64: one less their sum is what the teacher leaves to all others)
          P[s] = distill_exp(e64, lps);
          q[s] = te(yk[s] - high);
          near += (double)q[s];
          ek += distill_exp(e64, off);
          mass += P[s];
          if (P[s] != 0.0) a += P[s] * (lps - off);
        }
      }
    }
    if (bad) a = (double)NAN;
    all = wave_sum(all - near);  // the others: the very terms that the sum has of the teacher's tokens leave it
    ek = wave_sum(ek);
    mass = wave_sum(mass);
    a = wave_sum(a);
    float most = high;
    double sr = all, down = 1.0;
    if (!(all > ek * 0x1p-28)) {
      // (uniform) next to nothing is left: from the others' own maximum, the teacher's tokens masked
      float mz = -INFINITY;
      float rest = 0.f;
#pragma unroll
      for (int r = 0; r < VPT; ++r) {
        const int j = li + r * LANES;
        const uint32_t mask = j < vecs ? marks[j * N >> 5] >> (j * N & 31) : 0u;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (mask >> e & 1u) y[r][e] = -INFINITY;
          mz = fmaxf(mz, y[r][e]);
        }
      }
      mz = wave_most(mz);
      // (no other token: any finite stand-in, their sum is zero)
      most = mz == -INFINITY ? 0.f : mz;
#pragma unroll
      for (int r = 0; r < VPT; ++r)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x = te(y[r][e] - most);
          rest += x;
          if (CAP && x != 0.f) {
            float unused;
            sl[r][e] = x * f.slope_any(tof(v[r].e[e]), unused);
          } else {
            sl[r][e] = x;
          }
        }
      sr = (double)wave_sum(rest);
      down = distill_exp(e64, ((double)most - (double)high) * p.inv_t);
    }
    const DistillFactors k = distill_factors(p, mass, a, sr, ek, down);
    if (li == rr) {
      mine = DistillTerms{mass, a, ek, (float)sr, 0.0};
      mine_w = w;
      mine_rest = k.rest;
      mine_mr = most;
      mine_hi = high;
      mine_inv = k.inv;
      mine_mass = k.mass;
    }
    if (rr + 1 < R && n + 1 < p.rows) in.gather(p, n + 1, zn);
    if constexpr (GRAD) {
      const float c = w * inv_t, cr = c * k.rest;
#pragma unroll
      for (int r = 0; r < VPT; ++r) {
        const int j = li + r * LANES;
        if (j >= vecs) continue;
        Vec16<E> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.e[e] = cvt<E>(sl[r][e] * cr);
        put(j, o);
      }
      // the teacher's tokens over those (a wave's stores keep their order)
      wave_lds_sync();
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (id[s] >= 0) out[id[s]] = cvt<E>(c * k.of_teacher(P[s], q[s]) * slk[s]);
    } else {
      wave_lds_sync();
    }
  }
  double term = 0.0;
  const int64_t n = row0 + li;
  if (li < R && n < p.rows) {
    mine.dm = ((double)mine_mr - (double)mine_hi) * p.inv_t;
    const double each = mine_w != 0.f ? distill_loss_of(p, mine) : 0.0;
    term = mine_w != 0.f ? each * (double)mine_w : 0.0;
    p.each[n] = (float)each;
    if (p.stats) {
      p.stats[n] = mine_mr;
      p.stats[p.rows + n] = mine_rest;
      p.stats[2 * p.rows + n] = mine_hi;
      p.stats[3 * p.rows + n] = mine_inv;
      p.stats[4 * p.rows + n] = mine_mass;
    }
  }
#pragma unroll
  for (int o = R / 2; o >= 1; o >>= 1) term += __shfl_xor(term, o, 64);
  if (li == 0) sums[gi] = term;
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int i = 0; i < GROUPS; ++i) total += sums[i];
    p.part[blockIdx.x] = total;
  }
}

// A row's gradient where no token is the teacher's: cr e^{x - maximum} slope, by LANES threads.
template <typename E, bool CAP, int LANES>
__device__ __forceinline__ void distill_others(const E* row, E* out, int V, const Logit<CAP>& f, float cr, const TemperedExp& te,
                                               float most, int li) {
  constexpr int N = Vec16<E>::N, U = 2;
  auto one = [&](float z) {
    float y;
    const float slope = f.slope_any(z, y);
    return te(y - most) * slope * cr;
  };
  // the output's vectors; where the logits' do not start with them, they are read element by element
  const RowSpan<E> to(out, V);
  const bool together = (((uintptr_t)(row + to.head)) & 15) == 0;
  for (int j0 = li; j0 < to.vecs; j0 += U * LANES) {
    Vec16<E> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * LANES;
      v[u].raw = make_uint4(0u, 0u, 0u, 0u);
      if (j >= to.vecs) continue;
      if (together)
        v[u].raw = ((const Vec16<E>*)(row + to.head))[j].raw;
      else
#pragma unroll
        for (int e = 0; e < N; ++e) v[u].e[e] = row[to.head + j * N + e];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * LANES;
      if (j >= to.vecs) continue;
      Vec16<E> o;
      if (f.some_far(v[u])) {
#pragma unroll
        for (int e = 0; e < N; ++e) o.e[e] = cvt<E>(one(tof(v[u].e[e])));
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float y = f.near(tof(v[u].e[e]));
          o.e[e] = cvt<E>(te(y - most) * f.slope_near(y) * cr);
        }
      }
      ((Vec16<E>*)(out + to.head))[j].raw = o.raw;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (li < to.head) out[li] = cvt<E>(one(tof(row[li])));
  for (int i = to.head + to.vecs * N + li; i < V; i += LANES) out[i] = cvt<E>(one(tof(row[i])));
}

// Longer rows, a workgroup each: a running maximum and sum, then the gradient from a second reading,
// which finds the row in the caches.
template <typename E, bool CAP, int THREADS, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_long_kernel(DistillP p) {
  constexpr int N = Vec16<E>::N, WAVES = THREADS / 64, U = 2;
  extern __shared__ uint32_t marks[];
  __shared__ double sm_a[WAVES], sm_mass[WAVES], sm_ek[WAVES];
  __shared__ float sm[4][WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = p.V, K = p.K;
  const int64_t n = blockIdx.x;
  const float w = p.w ? p.w[n] : 1.f / (float)p.rows;
  const E* row = (const E*)p.z + n * p.stride;
  E* out = GRAD ? (E*)p.dz + n * (int64_t)V : nullptr;
  const RowSpan<E> to(out, V);
  if (w == 0.f) {  // (uniform)
    if (GRAD) {
      Vec16<E> zero;
      zero.raw = make_uint4(0u, 0u, 0u, 0u);
      for (int j = tid; j < to.vecs; j += THREADS) ((Vec16<E>*)(out + to.head))[j].raw = zero.raw;
      if (tid < to.head) out[tid] = (E)0.f;
      for (int i = to.head + to.vecs * N + tid; i < V; i += THREADS) out[i] = (E)0.f;
    }
    if (tid == 0) {
      p.each[n] = 0.f;
      p.part[n] = 0.0;
      if (p.stats)
        for (int i = 0; i < 5; ++i) p.stats[i * p.rows + n] = 0.f;
    }
    return;
  }
  const int64_t* ids = p.ids + n * K;
  const float* lps = p.lps + n * K;
  const Logit<CAP> f(p.cap);
  const Exp64 e64{kPowers64};
  const float inv_t = (float)p.inv_t;
  // the teacher's tokens, a bit each (from the 16-byte boundary at or before the row's start), and
  // their highest logit
  const int shift = (int)(((uintptr_t)row & 15) / sizeof(E)), vecs = (V + shift + N - 1) / N;
  for (int i = tid; i < (vecs * N + 31) / 32; i += THREADS) marks[i] = 0;
  __syncthreads();
  bool bad = false;
  float hz = -INFINITY, hl = -INFINITY;
  for (int k = tid; k < K; k += THREADS) {
    const int64_t id = ids[k];
    if (id >= V) bad = true;
    if (id < 0 || id >= V) continue;
    const uint32_t bit = (uint32_t)(id + shift);
    bad |= atomicOr(&marks[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1u;
    hz = fmaxf(hz, tof(row[id]));
    hl = fmaxf(hl, lps[k]);
  }
  __syncthreads();
  // the others
  const TemperedExp te(p.inv_t);
  float most = kLowest, sr = 0.f;
  for (int j0 = tid; j0 < vecs; j0 += U * THREADS) {
    Vec16<E> v[U];
    uint32_t mask[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * THREADS, i0 = j * N - shift;
      mask[u] = 0xffu;
      v[u].raw = make_uint4(0u, 0u, 0u, 0u);
      if (j >= vecs) continue;
      mask[u] = marks[j * N >> 5] >> (j * N & 31) & ((1u << N) - 1u);
      if (i0 >= 0 && i0 + N <= V) {
        v[u].raw = *(const uint4*)(row + i0);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (i0 + e >= 0 && i0 + e < V)
            v[u].e[e] = row[i0 + e];
          else
            mask[u] |= 1u << e;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N], top = most;
      if (f.some_far(v[u])) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = f.any(tof(v[u].e[e]));
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = f.near(tof(v[u].e[e]));
      }
      if (mask[u]) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = mask[u] >> e & 1u ? -INFINITY : x[e];
      }
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, x[e]);
      sr *= te(most - top);
#pragma unroll
      for (int e = 0; e < N; ++e) sr += te(x[e] - top);
      most = top;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  {
    const float top = wave_most(most);
    sr = wave_sum(sr * te(most - top));
    hz = wave_most(hz);
    hl = wave_most(hl);
    if (lane == 0) {
      sm[0][wave] = top;
      sm[1][wave] = sr;
      sm[2][wave] = hz;
      sm[3][wave] = hl;
    }
    __syncthreads();
    most = kLowest;
#pragma unroll
    for (int u = 0; u < WAVES; ++u) {
      most = fmaxf(most, sm[0][u]);
      hz = fmaxf(hz, sm[2][u]);
      hl = fmaxf(hl, sm[3][u]);
    }
    if (p.tail) hl = 0.f;
    sr = 0.f;
#pragma unroll
    for (int u = 0; u < WAVES; ++u) sr = fmaf(sm[1][u], te(sm[0][u] - most), sr);
  }
  // (no other token: any finite stand-in, their sum is zero)
  if (sr == 0.f) most = 0.f;
  const float high = sr == 0.f ? f.any(hz) : fmaxf(most, f.any(hz));
  double mass = 0.0, a = 0.0, ek = 0.0;
  for (int k = tid; k < K; k += THREADS) {
    const int64_t id = ids[k];
    if (id < 0 || id >= V) continue;
    const double off = ((double)f.any(tof(row[id])) - (double)high) * p.inv_t, lp = (double)lps[k] - (double)hl;
    // (in fp64: one less their sum is what the teacher leaves to all others)
    const double P = distill_exp(e64, lp);
    ek += distill_exp(e64, off);
    mass += P;
    if (P != 0.0) a += P * (lp - off);
  }
  if (bad) a = (double)NAN;
  ek = wave_sum(ek);
  mass = wave_sum(mass);
  a = wave_sum(a);
  __syncthreads();
  if (lane == 0) {
    sm_ek[wave] = ek;
    sm_mass[wave] = mass;
    sm_a[wave] = a;
  }
  __syncthreads();
  mass = a = ek = 0.0;
#pragma unroll
  for (int u = 0; u < WAVES; ++u) {
    ek += sm_ek[u];
    mass += sm_mass[u];
    a += sm_a[u];
  }
  const double dm = ((double)most - (double)high) * p.inv_t;
  const DistillFactors k = distill_factors(p, mass, a, sr, ek, distill_exp(e64, dm));
  if (tid == 0) {
    const double each = distill_loss_of(p, DistillTerms{mass, a, ek, sr, dm});
    p.each[n] = (float)each;
    p.part[n] = each * (double)w;
    if (p.stats) {
      p.stats[n] = most;
      p.stats[p.rows + n] = k.rest;
      p.stats[2 * p.rows + n] = high;
      p.stats[3 * p.rows + n] = k.inv;
      p.stats[4 * p.rows + n] = k.mass;
    }
  }
  if constexpr (GRAD) {
    const float c = w * inv_t;
    distill_others<E, CAP, THREADS>(row, out, V, f, c * k.rest, te, most, tid);
    __threadfence_block();
    __syncthreads();
    for (int i = tid; i < K; i += THREADS) {
      const int64_t id = ids[i];
      if (id < 0 || id >= V) continue;
      float y;
      const float slope = f.slope_any(tof(row[id]), y);
      out[id] = cvt<E>(c * k.of_teacher(distill_exp(e64, (double)lps[i] - (double)hl), te(y - high)) * slope);
    }
  }
}

template <typename E, bool CAP, int LANES>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillP p) {
  constexpr int N = Vec16<E>::N, GROUPS = 256 / LANES;
  __shared__ double sm[4];
  const int tid = threadIdx.x, gi = tid / LANES, li = tid % LANES;
  const int64_t n = (int64_t)blockIdx.x * GROUPS + gi;
  if (n >= p.rows || (p.formed && p.g[0] == 1.f)) return;  // (a whole wave, or none of the workgroup)
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
  const Exp64 e64{kPowers64};
  const TemperedExp te(p.inv_t);
  const float c = w * p.g[0] * (float)p.inv_t, most = p.stats[n], high = p.stats[2 * p.rows + n];
  DistillFactors k;
  k.rest = p.stats[p.rows + n];
  k.inv = p.stats[3 * p.rows + n];
  k.mass = p.stats[4 * p.rows + n];
  k.norm = 1.f;
  distill_others<E, CAP, LANES>(row, out, V, f, c * k.rest, te, most, li);
  // the teacher's tokens over those
  double top = 0.0;
  auto share = [&](float lp) { return distill_exp(e64, (double)lp - top); };
  if (!p.tail) {
    float hl = -INFINITY;
    for (int i = li; i < p.K; i += LANES) {
      const int64_t id = p.ids[n * p.K + i];
      if (id >= 0 && id < V) hl = fmaxf(hl, p.lps[n * p.K + i]);
    }
    top = (double)team.most(hl);
    double sum = 0.0;
    for (int i = li; i < p.K; i += LANES) {
      const int64_t id = p.ids[n * p.K + i];
      if (id >= 0 && id < V) sum += share(p.lps[n * p.K + i]);
    }
    k.norm = rcp((float)team.sum(sum));
  }
  __threadfence_block();
  team.sync();
  for (int i = li; i < p.K; i += LANES) {
    const int64_t id = p.ids[n * p.K + i];
    if (id < 0 || id >= V) continue;
    float y;
    const float slope = f.slope_any(tof(row[id]), y);
    out[id] = cvt<E>(c * k.of_teacher(share(p.lps[n * p.K + i]), te(y - high)) * slope);
  }
}

}  // namespace ts

namespace {

using ts::DistillP;
using ts::fail;

bool by_wave(int V) { return V <= 2048; }

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
  p->aligned = d->aligned;
  if (d->aligned && (((uintptr_t)io->logits & 15u) || (d->rows > 1 && d->stride % (d->dtype == TS_BF16 ? 8 : 4))))
    return fail(TS_ERR_VALUE, "distill: rows that are not aligned");
  p->inv_t = 1.0 / d->temperature;
  p->z = io->logits; p->ids = io->ids; p->lps = io->log_probs; p->w = io->weights;
  p->each = io->each; p->stats = io->stats; p->part = io->parts;
  return TS_OK;
}


// Whether a wave holds a row in its registers, `per` logits a lane (an unaligned row begins up to a vector
// less one behind the boundary that they count from), and 256 of a teacher's tokens.
constexpr int kPer = 32;
bool fits(const DistillP& p, bool bf, int per) { return p.V + (p.aligned ? 0 : (bf ? 8 : 4) - 1) <= 64 * per; }
bool in_registers(const DistillP& p, bool bf) { return p.K <= 256 && fits(p, bf, kPer); }
// Rows of a wave: several (the next row's loads then hide behind a row's arithmetic), where there are enough to
// keep every CU busy all the same.  Loss and gradient in us, eight and one: 2048 rows of 1024 (K 32, capped)
// 35 and 18, 8192 41 and 44, 16384 50 and 76, 32768 80 and 136; of 2048 (K 64) 16384 59 and 55, 32768 128 and 112.
int rows_of(const DistillP& p) { return p.rows >= 16384 ? 8 : 1; }

int64_t blocks_of(const DistillP& p, bool bf) {
  if (!in_registers(p, bf)) return p.rows;
  const int per = 4 * rows_of(p);
  return (p.rows + per - 1) / per;
}

template <typename E, bool CAP, bool GRAD>
int forward(const DistillP& p, hipStream_t stream) {
  constexpr bool BF = sizeof(E) == 2;
  constexpr int VPT = kPer / (BF ? 8 : 4);
  const dim3 grid((unsigned)blocks_of(p, BF));
  if (in_registers(p, BF)) {
#define TS_ROWS(vpt, ks, r) \
  hipLaunchKernelGGL((ts::distill_rows_kernel<E, CAP, vpt, ks, r, GRAD>), grid, dim3(256), 0, stream, p)
    if (rows_of(p) == 1)
      TS_ROWS(VPT, 4, 1);
    else if (p.K > 64)
      TS_ROWS(VPT, 4, 8);
    else if (fits(p, BF, kPer / 2))
      TS_ROWS(VPT / 2, 1, 8);
    else
      TS_ROWS(VPT, 1, 8);
#undef TS_ROWS
    return TS_OK;
  }
  const int lds = ((p.V + 15) / 32 + 2) * 4;
  // (1024 threads a row and 256, K 64: 256 rows of 32768 23 and 28 us, 512 38 and 34, 4096 241 and 180; of 5000
  // 256 rows 16 and 14, 4096 138 and 46)
  const bool few = p.rows < 512;
  const void* fn = few ? (const void*)ts::distill_long_kernel<E, CAP, 1024, GRAD>
                       : (const void*)ts::distill_long_kernel<E, CAP, 256, GRAD>;
  const hipError_t e = ts::ensure_lds_limit(fn, (1 << 17) + 8);
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "distill: %s", hipGetErrorString(e));
  if (few)
    hipLaunchKernelGGL((ts::distill_long_kernel<E, CAP, 1024, GRAD>), grid, dim3(1024), lds, stream, p);
  else
    hipLaunchKernelGGL((ts::distill_long_kernel<E, CAP, 256, GRAD>), grid, dim3(256), lds, stream, p);
  return TS_OK;
}
template <typename E>
int forward(const DistillP& p, hipStream_t stream) {
  if (p.cap == 0.f) return p.dz ? forward<E, false, true>(p, stream) : forward<E, false, false>(p, stream);
  return p.dz ? forward<E, true, true>(p, stream) : forward<E, true, false>(p, stream);
}

template <typename E, bool CAP>
int backward(const DistillP& p, hipStream_t stream) {
  const dim3 grid((unsigned)(by_wave(p.V) ? (p.rows + 3) / 4 : p.rows));
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

int ts_distill_fwd(const ts_distill_desc* d, const ts_distill_io* io, hipStream_t stream) {
  DistillP p;
  int rc = setup(d, io, &p);
  if (rc) return rc;
  if (!io->loss || (d->rows && (!io->each || !io->parts))) return fail(TS_ERR_VALUE, "distill: missing tensors");
  p.dz = io->dlogits;
  const bool bf = d->dtype == TS_BF16;
  if (p.dz && ((uintptr_t)p.dz & 15u)) return fail(TS_ERR_VALUE, "distill: misaligned gradient");
  if (d->rows) {
    rc = bf ? forward<ts::bf16>(p, stream) : forward<float>(p, stream);
    if (rc) return rc;
  }
  hipLaunchKernelGGL(ts::rows_sum_kernel, dim3(1), dim3(1024), 0, stream, (const double*)io->parts,
                     d->rows ? blocks_of(p, bf) : 0, io->loss);
  return finish("distill");
}

static int distill_bwd(const ts_distill_desc* d, const ts_distill_io* io, const float* dloss, void* dlogits, bool formed,
                       hipStream_t stream) {
  DistillP p;
  int rc = setup(d, io, &p);
  if (rc || d->rows == 0) return rc;
  if (!io->stats || !dloss || !dlogits || ((uintptr_t)dlogits & (d->dtype == TS_BF16 ? 1u : 3u)))
    return fail(TS_ERR_VALUE, "distill bwd: missing or misaligned tensors");
  p.g = dloss;
  p.dz = dlogits;
  p.formed = formed;
  if (d->dtype == TS_BF16)
    rc = d->cap == 0.f ? backward<ts::bf16, false>(p, stream) : backward<ts::bf16, true>(p, stream);
  else
    rc = d->cap == 0.f ? backward<float, false>(p, stream) : backward<float, true>(p, stream);
  return rc ? rc : finish("distill bwd");
}

int ts_distill_bwd(const ts_distill_desc* d, const ts_distill_io* io, const float* dloss, void* dlogits,
                   hipStream_t stream) {
  return distill_bwd(d, io, dloss, dlogits, false, stream);
}

int ts_distill_scale(const ts_distill_desc* d, const ts_distill_io* io, const float* dloss, hipStream_t stream) {
  return distill_bwd(d, io, dloss, io ? io->dlogits : nullptr, true, stream);
}

}  // extern "C"
