// Sampling of tokens from (soft-capped) logits with temperature, top-k, top-p and min-p, from
// given random numbers (gfx950).
//
//   y = cap tanh(z / cap) (or z);  w_i = round(2^44 e^{(y_i - max y) / temperature})
//   left: the top_k highest logits (ties: the lowest index first); of those, in that order, while the
//   weight before a token is less than top_p of theirs; of those, w_i >= min_p 2^44
//   token: the first, by index, whose running weight is over floor(u total)
//
// The weights are whole numbers, so that their sums are the same in any order: what is left, and
// the token, do not depend on how the work is split.  They come from an exponential in fp64.
//
// A workgroup takes a row.  A cut (of top-k by counts, of top-p by weights) is found without
// sorting: a histogram over the distance from the maximum, in LDS by integer atomics, then
// histograms of the keys inside the bin that the cut falls into, down to one key, then of
// the indices of its ties.  The token is found the same way, by weights over the indices.  Few tokens
// or a small nucleus are sorted in LDS instead.  256 rows of 131072 logits, settings a row: 160 us, bound by
// the passes over a row that one CU makes, two of them with fp64 exponentials.

#include "ts_common.h"
#include "ts_logits.h"
#include "ts_tokens.h"

#include <string.h>

namespace ts {

typedef unsigned long long u64;

struct SampleP {
  int64_t rows, stride;
  int V;
  float cap;
  double temperature, top_p, min_p;
  int64_t top_k;
  const void* z;
  const float* u;
  const float *temperatures, *top_ps, *min_ps;
  const int64_t* top_ks;
  int64_t* tokens;
  float* log_probs;
};

constexpr int kBins = 2048;
constexpr int kList = 2048;  // tokens that are sorted at once
constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr float kSpan = 31.3f;              // e^-kSpan 2^44 < 1 / 2: weights beyond it are zero

// Keys in the order of their logits (-0 as 0).
template <typename E> struct KeyOf;
template <> struct KeyOf<float> {
  static __device__ __forceinline__ uint32_t key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
  }
};
template <> struct KeyOf<bf16> {
  static __device__ __forceinline__ uint32_t key(float x) { return KeyOf<float>::key(x) >> 16; }
  static __device__ __forceinline__ float value(uint32_t k) {
    return KeyOf<float>::value(k & 0x8000u ? k << 16 : k << 16 | 0xffffu);
  }
};

template <typename E, bool CAP, int THREADS>
struct Sampler {
  static constexpr int N = Vec16<E>::N, WAVES = THREADS / 64;
  struct Shared {
    u64 bins[kBins];
    u64 list[kList];
    u64 sums[WAVES];
    double table[64];
    float most[WAVES], total[WAVES], high[WAVES];
    u64 before, inside;
    int at, count, token;
  };
  Shared& sh;
  const SampleP& p;
  const E* row;
  const Vec16<E>* vec;
  int V, shift, vecs, tid, lane, wave;
  Exp64 e64;
  float most;         // the highest logit
  double base;        // see logit()
  double top, inv_t;  // as the softmax takes it, and one over the temperature
  float scale;        // bins of a unit of logits
  uint32_t cut_key, cut_index;  // left: keys above, and that key before the index
  u64 least;                    // and weights of at least this

  __device__ __forceinline__ Sampler(Shared& s, const SampleP& q) : sh(s), p(q) {
    tid = threadIdx.x;
    lane = tid & 63;
    wave = tid >> 6;
    V = p.V;
    row = (const E*)p.z + (int64_t)blockIdx.x * p.stride;
    shift = (int)(((uintptr_t)row & 15) / sizeof(E));
    vec = (const Vec16<E>*)(row - shift);
    vecs = (V + shift + N - 1) / N;
    e64.table = sh.table;
    if (tid < 64) sh.table[tid] = kPowers64[tid];
    cut_key = 0;
    cut_index = 0xffffffffu;
    least = 1;
  }

  // A vector of the row; what lies before its start or behind its end is not read and stands as -inf.
  __device__ __forceinline__ Vec16<E> load(int j) const {
    Vec16<E> v;
    const int i0 = j * N - shift;
    if (i0 >= 0 && i0 + N <= V) {
      v.raw = vec[j].raw;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v.e[e] = (E)-INFINITY;
        if (i0 + e >= 0 && i0 + e < V) v.e[e] = row[i0 + e];
      }
    }
    return v;
  }
  // f(vector's number, its elements) of every vector (what lies past the row's ends stands as -inf), four
  // on their way at once, one copy of f's code
  template <typename F>
  __device__ __forceinline__ void vectors(F f) const {
#pragma unroll 1
    for (int j = tid; j < vecs; j += 4 * THREADS) {
      Vec16<E> a = load(j), b, c, d;
      if (j + THREADS < vecs) b = load(j + THREADS);
      if (j + 2 * THREADS < vecs) c = load(j + 2 * THREADS);
      if (j + 3 * THREADS < vecs) d = load(j + 3 * THREADS);
#pragma unroll 1
      for (int i = j; i < min(vecs, j + 4 * THREADS); i += THREADS) {
        f(i, a);
        a.raw = b.raw;
        b.raw = c.raw;
        c.raw = d.raw;
      }
    }
  }
  // f(logit, index) of a vector's elements
  template <typename F>
  __device__ __forceinline__ void elements(int j, const Vec16<E>& v, F f) const {
#pragma unroll
    for (int e = 0; e < N; ++e) f(tof(v.e[e]), j * N - shift + e);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    vectors([&](int j, const Vec16<E>& v) { elements(j, v, f); });
  }

  // A logit as the softmax takes it, in fp64, less `base`: the cap where the highest logit is near it
  // (their distance from the cap, -2 cap / (1 + e^{2 z / cap}), has the digits there), else
  // zero.  Below a quarter of the cap tanh is a ratio of polynomials (its continued fraction's sixth
  // step, off by 2^-54).
  __device__ __forceinline__ double logit(float x) const {
#pragma clang fp contract(off)
    if (!CAP) return (double)x;
    const double c = (double)p.cap, a = fmin(fabs((double)x) / c, 300.0);
    if (a < 0.25) {
      const double t = (double)x / c, u = t * t;
      const double n = fma(fma(21.0, u, 1260.0), u, 10395.0), d = fma(fma(u + 210.0, u, 4725.0), u, 10395.0);
      return c * (t * n / d) - base;
    }
    const double e = e64(-2.0 * a);
    return (c - base) - 2.0 * c * ((x > 0.f ? e : 1.0) / (1.0 + e));
  }
  __device__ __forceinline__ u64 weight(float x) const {
#pragma clang fp contract(off)
    if (x == most) return (u64)kUnit;
    if (CAP ? x == -INFINITY : (x - most) * (float)inv_t < -(kSpan + 1.f)) return 0;
    const double t = (logit(x) - top) * inv_t;
    if (!(t > -(double)kSpan)) return 0;
    return e64.whole(t);
  }
  __device__ __forceinline__ bool left(float x, int i) const {
    const uint32_t k = KeyOf<E>::key(x);
    return k > cut_key || (k == cut_key && (uint32_t)i < cut_index);
  }
  __device__ __forceinline__ int bin_of(float x) const { return (int)fminf((most - x) * scale, (float)(kBins - 1)); }

  __device__ __forceinline__ void clear() {
    __syncthreads();
    for (int i = tid; i < kBins; i += THREADS) sh.bins[i] = 0;
    __syncthreads();
  }
  // The first bin that ok(what comes before it) holds for and ok(what comes before the next) does
  // not; -1 if there is none.  `before` is what comes before the bins, and then before that bin.
  template <typename OK>
  __device__ __forceinline__ int find(u64& before, u64& inside, OK ok) {
    constexpr int PER = kBins / THREADS;
    __syncthreads();
    if (tid == 0) sh.at = -1;
    u64 own[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += own[i] = sh.bins[tid * PER + i];
    u64 run = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 x = __shfl_up(run, o, 64);
      if (lane >= o) run += x;
    }
    if (lane == 63) sh.sums[wave] = run;
    __syncthreads();
    u64 at = before + run - sum;
    for (int w = 0; w < wave; ++w) at += sh.sums[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (ok(at) && !ok(at + own[i])) {
        sh.at = tid * PER + i;
        sh.before = at;
        sh.inside = own[i];
      }
      at += own[i];
    }
    __syncthreads();
    if (sh.at >= 0) {
      before = sh.before;
      inside = sh.inside;
    }
    return sh.at;
  }
  static __device__ __forceinline__ int bits_over(uint32_t range, int bits) {  // range >> this < 2^bits
    return range >> bits ? 32 - bits - __builtin_clz(range) : 0;
  }

  // Cuts what is left to the tokens with ok(measure of those before it), in the order of logits.
  template <typename M, typename OK>
  __device__ __forceinline__ void cut(M measure, OK ok) {
    clear();
    each([&](float x, int i) {
      const u64 w = left(x, i) ? measure(x) : 0;
      if (w) atomicAdd(&sh.bins[bin_of(x)], w);
    });
    u64 before = 0, inside = 0;
    const int b = find(before, inside, ok);
    if (b < 0) return;
    // keys that the bin's logits have at most: its ends, and what their rounding may be off
    const float far = (float)(b + 1) / scale, slack = 1e-6f * (fabsf(most) + far);
    uint32_t hi = KeyOf<E>::key(fminf(most, most - (float)b / scale + slack));
    uint32_t lo = b == kBins - 1 ? KeyOf<E>::key(-INFINITY) : KeyOf<E>::key(most - far - slack);
    for (;;) {
      const int s = bits_over(hi - lo, 11);
      clear();
      each([&](float x, int i) {
        const uint32_t k = KeyOf<E>::key(x);
        if (k < lo || k > hi || bin_of(x) != b || !left(x, i)) return;
        const u64 w = measure(x);
        if (w) atomicAdd(&sh.bins[(hi - k) >> s], w);
      });
      const int at = find(before, inside, ok);
      if (at < 0) return;  // (every key of the bin lies between lo and hi)
      const uint32_t h = hi - ((uint32_t)at << s), span = (1u << s) - 1u;
      hi = h;
      lo = h - lo > span ? h - span : lo;
      if (!s) break;
    }
    // one key; as many of its ties as ok allows
    const u64 one = measure(KeyOf<E>::value(hi));
    u64 some = 1, most_ties = inside / one;
    const u64 ties = most_ties;
    while (some < most_ties) {  // the least `some` with ok false behind it
      const u64 half = (some + most_ties) / 2;
      if (ok(before + half * one))
        some = half + 1;
      else
        most_ties = half;
    }
    const uint32_t key = hi;
    uint32_t limit = 0xffffffffu;
    if (some < ties) {
      uint32_t i0 = 0, i1 = (uint32_t)V - 1;
      u64 n = 0;
      for (;;) {
        const int s = bits_over(i1 - i0, 11);
        clear();
        each([&](float x, int i) {
          if (KeyOf<E>::key(x) == key && left(x, i) && (uint32_t)i >= i0 && (uint32_t)i <= i1)
            atomicAdd(&sh.bins[((uint32_t)i - i0) >> s], (u64)1);
        });
        const int at = find(n, inside, [&](u64 c) { return c < some; });
        if (at < 0) return;
        const uint32_t a = i0 + ((uint32_t)at << s);
        i1 = min(i1, a + (1u << s) - 1u);
        i0 = a;
        if (!s) break;
      }
      limit = i0 + 1;
    }
    cut_index = key == cut_key ? min(limit, cut_index) : limit;
    cut_key = key;
  }

  __device__ __forceinline__ u64 block_sum(u64 x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
    __syncthreads();
    if (lane == 0) sh.sums[wave] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < WAVES; ++w) x += sh.sums[w];
    return x;
  }
  __device__ __forceinline__ u64 weights_left() {
    u64 sum = 0;
    each([&](float x, int i) {
      if (left(x, i)) sum += weight(x);
    });
    return block_sum(sum);
  }

  // ---- a list of tokens in LDS: key << 32 | ~index sorts them as the logits are ordered (from the top)
  static __device__ __forceinline__ u64 entry(uint32_t key, int i) { return (u64)key << 32 | (uint32_t)~(uint32_t)i; }
  static __device__ __forceinline__ uint32_t key_of(u64 x) { return (uint32_t)(x >> 32); }
  static __device__ __forceinline__ uint32_t index_of(u64 x) { return ~(uint32_t)x; }
  __device__ __forceinline__ void add_to_list(float x, int i) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kList) sh.list[at] = entry(KeyOf<E>::key(x), i);
  }
  // Sorts the list's first n, the highest first; `size`, a power of two from n on, is filled up with zeros.
  __device__ __forceinline__ void sort_list(int n) {
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += THREADS) sh.list[i] = 0;
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        __syncthreads();
        for (int i = tid; i < size / 2; i += THREADS) {
          const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
          const u64 a = sh.list[lo], b = sh.list[hi];
          if ((a < b) == ((lo & k) == 0)) {
            sh.list[lo] = b;
            sh.list[hi] = a;
          }
        }
      }
    __syncthreads();
  }
  // f(i, what comes before i) with the running sum of g(i) over the first n, from `before`; every thread
  // has a stretch of them.  Gives the whole sum.
  template <typename G, typename F>
  __device__ __forceinline__ u64 running(int n, u64 before, G g, F f) {
    constexpr int PER = kList / THREADS;
    const int per = (n + THREADS - 1) / THREADS;
    u64 own[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = tid * per + i;
      own[i] = i < per && at < n ? g(at) : 0;
      sum += own[i];
    }
    u64 run = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 x = __shfl_up(run, o, 64);
      if (lane >= o) run += x;
    }
    __syncthreads();
    if (lane == 63) sh.sums[wave] = run;
    __syncthreads();
    u64 at = before + run - sum, all = 0;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) at += sh.sums[w];
      all += sh.sums[w];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = tid * per + i;
      if (i < per && k < n) f(k, at, own[i]);
      at += own[i];
    }
    return all;
  }
  __device__ __forceinline__ u64 list_weight(int i) const { return weight(KeyOf<E>::value(key_of(sh.list[i]))); }

  // floor(u total), below the total
  static __device__ __forceinline__ u64 place_of(double u, u64 total) {
    const double place = floor((u > 0.0 ? u : 0.0) * (double)total);
    return place >= (double)total ? total - 1 : (u64)place;
  }

  // The token where everything that is left stands in the list's first n (sorted): the nucleus among them, the
  // least share, then the running weights in the order of the indices.
  __device__ __forceinline__ int pick_of_list(int n, double top_p, double u) {
    if (top_p < 1.0) {
      const u64 all = running(n, 0, [&](int i) { return list_weight(i); }, [](int, u64, u64) {});
      const double part = top_p * (double)all;
      __syncthreads();
      if (tid == 0) sh.at = n;
      __syncthreads();
      running(n, 0, [&](int i) { return list_weight(i); }, [&](int i, u64 before, u64) {
        if (before != 0 && !((double)before < part)) atomicMin(&sh.at, i);
      });
      __syncthreads();
      n = sh.at;
    }
    // (in the order of their indices: the key goes behind the index)
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      const u64 x = sh.list[i];
      sh.list[i] = (u64)(uint32_t)x << 32 | key_of(x);  // ~index: the lowest index is the highest
    }
    __syncthreads();
    sort_list(n);
    auto w = [&](int i) {
      const u64 x = weight(KeyOf<E>::value((uint32_t)sh.list[i]));
      return x >= least ? x : 0;
    };
    const u64 want = place_of(u, running(n, 0, w, [](int, u64, u64) {}));
    __syncthreads();
    if (tid == 0) sh.at = 0;
    __syncthreads();
    running(n, 0, w, [&](int i, u64 before, u64 own) {
      if (before <= want && before + own > want) sh.at = i;
    });
    __syncthreads();
    return (int)~(uint32_t)(sh.list[sh.at] >> 32);
  }

  // The token by the weights over the vectors that stand in the bins (2^sv vectors each), their sum total.
  __device__ __forceinline__ int pick_of_bins(int sv, u64 total, double u) {
    const u64 want = place_of(u, total);
    u64 before = 0, inside;
    const int b = find(before, inside, [&](u64 c) { return c <= want; });
    // (the bin's elements; one wave, each lane the next one in turn)
    if (wave == 0) {
      const int i0 = ((b << sv) * N) - shift, i1 = min(V, i0 + (N << sv));
      int found = -1;
      for (int at = max(i0, 0); at < i1 && found < 0; at += 64) {
        const int i = at + lane;
        u64 w = 0;
        if (i < i1) {
          const float x = tof(row[i]);
          if (left(x, i)) w = weight(x);
          if (w < least) w = 0;
        }
        u64 run = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const u64 x = __shfl_up(run, o, 64);
          if (lane >= o) run += x;
        }
        const u64 mask = __ballot(before + run > want);
        if (mask)
          found = at + __builtin_ctzll(mask);
        else
          before += __shfl(run, 63, 64);
      }
      if (lane == 0) sh.token = max(found, 0);
    }
    __syncthreads();
    return sh.token;
  }
  // Adds the weights of what is left to the bins of their vectors; gives the sum.
  __device__ __forceinline__ u64 fill_bins(int sv) {
    clear();
    u64 sum = 0;
    vectors([&](int j, const Vec16<E>& v) {
      u64 ws = 0;
      elements(j, v, [&](float x, int i) {
        if (left(x, i)) {
          const u64 w = weight(x);
          ws += w >= least ? w : 0;
        }
      });
      if (ws) atomicAdd(&sh.bins[j >> sv], ws);
      sum += ws;
    });
    return block_sum(sum);
  }

  __device__ __forceinline__ int pick(int64_t top_k, double top_p, double u, float mine) {
    const int sv = bits_over((uint32_t)(vecs - 1), 11);
    // (a list of them or cut after cut, 64 rows in us: 131072 logits, top_k 20 44 either way, 100 48 and 96, 500 64
    // and 103, past kList / 4 900 132 and 108; 32768, 500 43 and 44, 900 54 and 46; short rows' lists overflow
    // from 100 on: 8192, 250 56 and 30; 1024, 250 33 and 16)
    if (top_k < V && top_k <= kList / 4) {
      // The k-th highest of the threads' maxima bounds the k-th logit from below: what lies in its bin and
      // above is little more than k
      const u64 k = (u64)(top_k < 1 ? 1 : top_k);
      clear();
      if (mine > -INFINITY) atomicAdd(&sh.bins[bin_of(mine)], (u64)1);
      if (tid == 0) sh.count = 0;
      u64 before = 0, inside;
      int b = find(before, inside, [&](u64 c) { return c < k; });
      if (b < 0) b = kBins - 1;
      each([&](float x, int i) {
        if (x > -INFINITY && bin_of(x) <= b) add_to_list(x, i);
      });
      __syncthreads();
      const int n = sh.count;
      if (n <= kList) {
        __syncthreads();
        sort_list(n);
        return pick_of_list(min(n, (int)k), top_p, u);
      }
    } else if (top_k >= V && top_p < 1.0) {
      // weights by their distance from the maximum; the bin of the cut is sorted
      clear();
      if (tid == 0) sh.count = 0;
      u64 sum = 0, before = 0, inside;
      each([&](float x, int) {
        const u64 w = weight(x);
        if (w) atomicAdd(&sh.bins[bin_of(x)], w);
        sum += w;
      });
      const double part = top_p * (double)block_sum(sum);
      auto ok = [&](u64 c) { return c == 0 || (double)c < part; };
      const int b = find(before, inside, ok);
      if (b < 0) return pick_of_bins(sv, fill_bins(sv), u);
      // a small nucleus is sorted whole
      each([&](float x, int i) {
        if (bin_of(x) <= b && x > -INFINITY) add_to_list(x, i);
      });
      __syncthreads();
      const int held = sh.count;
      if (held <= kList) {
        __syncthreads();
        sort_list(held);
        if (tid == 0) sh.at = held;
        __syncthreads();
        running(held, 0, [&](int i) { return list_weight(i); }, [&](int i, u64 c, u64) {
          if (!ok(c)) atomicMin(&sh.at, i);
        });
        __syncthreads();
        return pick_of_list(sh.at, 1.0, u);
      }
      clear();
      if (tid == 0) sh.count = 0;
      __syncthreads();
      sum = 0;
      vectors([&](int j, const Vec16<E>& v) {
        u64 ws = 0;
        elements(j, v, [&](float x, int i) {
          const int at = bin_of(x);
          if (at > b || x == -INFINITY) return;
          if (at == b) {
            add_to_list(x, i);
          } else {
            const u64 w = weight(x);
            ws += w >= least ? w : 0;
          }
        });
        if (ws) atomicAdd(&sh.bins[j >> sv], ws);
        sum += ws;
      });
      __syncthreads();
      const int n = sh.count;
      if (n <= kList) {
        sum = block_sum(sum);
        sort_list(n);
        // the first of the list that is cut, and the weights of those before it
        __syncthreads();
        if (tid == 0) sh.at = n;
        __syncthreads();
        running(n, before, [&](int i) { return list_weight(i); }, [&](int i, u64 c, u64) {
          if (!ok(c)) atomicMin(&sh.at, i);
        });
        __syncthreads();
        const int m = sh.at;  // (one at least: ok holds before the bin)
        u64 more = 0;
        for (int i = tid; i < m; i += THREADS) {
          const u64 w = list_weight(i);
          if (w < least) continue;
          atomicAdd(&sh.bins[((int)index_of(sh.list[i]) + shift) / N >> sv], w);
          more += w;
        }
        const u64 last = sh.list[m - 1];
        cut_key = key_of(last);
        cut_index = index_of(last) + 1;
        return pick_of_bins(sv, sum + block_sum(more), u);
      }
    }
    // any other: cut after cut
    if (top_k < V) {
      const u64 k = top_k < 1 ? 1 : (u64)top_k;
      cut([&](float x) { return (u64)(x > -INFINITY); }, [&](u64 before) { return before < k; });
    }
    if (top_p < 1.0) {
      const double part = top_p * (double)weights_left();
      cut([&](float x) { return weight(x); }, [&](u64 before) { return before == 0 || (double)before < part; });
    }
    return pick_of_bins(sv, fill_bins(sv), u);
  }

  __device__ __forceinline__ void run() {
    const int64_t n = blockIdx.x;
    double temperature = p.temperatures ? (double)p.temperatures[n] : p.temperature;
    const double top_p = p.top_ps ? (double)p.top_ps[n] : p.top_p;
    const double min_p = p.min_ps ? (double)p.min_ps[n] : p.min_p;
    int64_t top_k = p.top_ks ? p.top_ks[n] : p.top_k;
    const double u = (double)p.u[n];
    // the highest logit, and the sum of e^{y - max} (fp32); a row with no logit, or with one that is no number or
    // +inf, has no token
    const Logit<CAP> f(p.cap);
    float mine = -INFINITY, ym = kLowest, s = 0.f;
    bool bad = !(temperature >= 0.0) || top_p != top_p || min_p != min_p;
    vectors([&](int, const Vec16<E>& v) {
      float y[N], top = ym;
      const bool far = f.some_far(v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x = tof(v.e[e]);
        mine = fmaxf(mine, x);
        bad |= !(x < INFINITY);
        y[e] = CAP && x == -INFINITY ? -INFINITY : far ? f.any(x) : f.near(x);
        top = fmaxf(top, y[e]);
      }
      s *= ex(ym - top);
#pragma unroll
      for (int e = 0; e < N; ++e) s += ex(y[e] - top);
      ym = top;
    });
    float hi = mine;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor(hi, o, 64));
      const float y2 = __shfl_xor(ym, o, 64), s2 = __shfl_xor(s, o, 64), top = fmaxf(ym, y2);
      s = s * ex(ym - top) + s2 * ex(y2 - top);
      ym = top;
    }
    if (lane == 0) {
      sh.most[wave] = hi;
      sh.high[wave] = ym;
      sh.total[wave] = s;
    }
    bad = __syncthreads_or(bad);
    most = -INFINITY;
    ym = kLowest;
    for (int w = 0; w < WAVES; ++w) {
      most = fmaxf(most, sh.most[w]);
      ym = fmaxf(ym, sh.high[w]);
    }
    if (bad || most == -INFINITY) {
      if (tid == 0) {
        p.tokens[n] = -1;
        p.log_probs[n] = NAN;
      }
      return;
    }
    s = 0.f;
    for (int w = 0; w < WAVES; ++w) s = fmaf(sh.total[w], ex(sh.high[w] - ym), s);

    if (temperature == 0.0) {  // the highest logit
      temperature = 1.0;
      top_k = 1;
    }
    inv_t = 1.0 / temperature;
    base = CAP && !(fabsf(most) < 0.25f * p.cap) ? (double)p.cap : 0.0;
    top = logit(most);
    scale = (float)fmin((double)kBins / ((double)kSpan * fmin(temperature, 1e30)), 1e30);
    if (min_p > 0.0) {
      const double w = ceil(fmin(min_p, 1.0) * kUnit);
      least = w > 1.0 ? (u64)w : 1;
    }
    const int token = pick(top_k, top_p, u, mine);
    if (tid == 0) {
      const float x = tof(row[token]);
      // (as of the fp32 maximum that the sum is taken from)
      const double off = f.any(x) >= ym ? 0.0 : logit(x) + base - (double)ym;
      p.tokens[n] = token;
      p.log_probs[n] = (float)(off - log((double)s));
    }
  }
};

template <typename E, bool CAP, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleP p) {
  typedef Sampler<E, CAP, THREADS> S;
  __shared__ typename S::Shared sh;
  S s(sh, p);
  __syncthreads();
  s.run();
}

}  // namespace ts

namespace {

using ts::fail;
using ts::SampleP;

template <typename E, bool CAP>
void launch(const SampleP& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.rows);
  // (256 and 1024 threads a row, a nucleus in us: 1024 logits, 16 rows 22 and 27, 1024 rows 28 and 100; 8192, 40 and
  // 37, 71 and 146; 16384, 70 and 49, 100 and 195; 32768, 133 and 71, 188 and 280)
  if (p.V <= 8192)
    hipLaunchKernelGGL((ts::sample_kernel<E, CAP, 256>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((ts::sample_kernel<E, CAP, 1024>), grid, dim3(1024), 0, stream, p);
}

}  // namespace

extern "C" {

int ts_sample_tokens(const ts_sample_desc* d, const ts_sample_io* io, hipStream_t stream) {
  if (!d || !io || d->rows < 0 || d->V < 1 || d->stride < 0 || !(d->cap == 0.f || (d->cap >= 1e-30f && d->cap <= 1e30f)) ||
      !(d->temperature >= 0.0) || !(d->top_p >= 0.0) || !(d->min_p >= 0.0) || d->top_k < 1)
    return fail(TS_ERR_VALUE, "sample: bad shape, cap, temperature, top_k, top_p or min_p");
  if (d->dtype != TS_BF16 && d->dtype != TS_F32) return fail(TS_ERR_NOT_IMPLEMENTED, "sample: bf16 or fp32 only");
  // (sums of weights stay in 63 bits; a launch counts its threads in 32)
  if (d->V >= 1 << 19) return fail(TS_ERR_NOT_IMPLEMENTED, "sample: fewer than 2^19 tokens, got %d", d->V);
  if (d->rows >= 1 << 22) return fail(TS_ERR_NOT_IMPLEMENTED, "sample: too many rows");
  if (d->rows == 0) return TS_OK;
  if (!io->logits || ((uintptr_t)io->logits & (d->dtype == TS_BF16 ? 1u : 3u)) || !io->uniforms || !io->tokens ||
      !io->log_probs)
    return fail(TS_ERR_VALUE, "sample: missing or misaligned tensors");
  SampleP p;
  memset(&p, 0, sizeof(p));
  p.rows = d->rows; p.stride = d->stride; p.V = d->V; p.cap = d->cap;
  p.temperature = d->temperature; p.top_p = d->top_p; p.min_p = d->min_p; p.top_k = d->top_k;
  p.z = io->logits; p.u = io->uniforms;
  p.temperatures = io->temperatures; p.top_ks = io->top_ks; p.top_ps = io->top_ps; p.min_ps = io->min_ps;
  p.tokens = io->tokens; p.log_probs = io->log_probs;
  if (d->dtype == TS_BF16)
    d->cap == 0.f ? launch<ts::bf16, false>(p, stream) : launch<ts::bf16, true>(p, stream);
  else
    d->cap == 0.f ? launch<float, false>(p, stream) : launch<float, true>(p, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "sample: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}

}  // extern "C"
