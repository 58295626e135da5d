// Windowed softmax attention with sinks, backward (gfx950).
//
// With P = 2^(scale2 q k - lse), dP = dout v^T and D = rowsum(dout out):
//   dS = P (dP - D),  dv = P^T dout,  dk = scale dS^T q,  dq = scale dS k
//
// The scores are formed again, from q, k and the forward's lse.  Two kernels: one owns
// queries (dq, and D, which the other reads), one owns keys (dk and dv, over the query heads
// that share them, so that their sums have a fixed order).  Each wave keeps the rows that it
// owns as MFMA operands and accumulates in fp32; what it walks over is staged in LDS once
// for both of its uses, by rows and by columns.  In bf16, P and dS enter the keys' products
// in bf16 (2^-9 of each, as the gradients' own rounding); the queries' takes dS in two parts: a
// query's dS add to zero, so that of keys that are alike little is left but what rounding leaves.
// At B8 H8 T4096 (64-wide on 4 key heads, window 1024) the keys' kernel takes 219 us and the queries' 170, the
// matrix cores busy in 24 and 31 % of them, other vector instructions in 20 and 40; at 16384 tokens of 8
// 128-wide heads 439 and 302 us, busy in 25 and 36 %: one tile in LDS with two barriers, not either unit, bounds
// the keys'.
//
// A sink is seen by every query behind its window: those pairs go to workgroups of their
// own, a stretch of queries each, which leave sums of the sinks' rows in fp32; where workgroups are
// few, the query heads that share a key head have workgroups (and sums) of their own.  A third
// kernel adds the sums in order.  In bf16, D takes out with what its rounding left of it.
//
// A hidden pair's zero times a key or a query that is not finite would be no number: where a workgroup's
// sums are not finite, it goes over its tiles again and adds only the pairs that there are, as the forward.

#include "ts_window.h"

#include <string.h>
#include <type_traits>

namespace ts {

int window_setup(const ts_window_desc* d, const ts_window_io* io, WinP* p);
int window_rows(const ts_strided& s, int vec);
bool window_narrow(const WinP& p, int B, bool bf, int heads);

// Whether a lane's sums are not all finite (a sum of magnitudes is where all are, or where none is near
// the border of its type).
template <int N, int DB>
__device__ __forceinline__ bool win_odd(const floatx4 (&acc)[N][DB]) {
  bool odd = false;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float all = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) all += fabsf(acc[n][db][i]);
    odd |= !(all < INFINITY);
  }
  return odd;
}

// A wave owns 16 NQ queries.
template <typename E, int D, int NQ>
__global__ __launch_bounds__(256, sizeof(E) == 2 ? (D == 64 ? 3 : 2) : 1) void window_dq_kernel(WinP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  constexpr int P = win_pitch<E, D>(), DB = D / 16, KB = D / 32, WQ = 16 * NQ, QT = 4 * WQ;
  extern __shared__ __align__(16) unsigned char lds[];
  E* kt = (E*)lds;  // [TT * P]
  E* vt = kt + TT * P;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * QT, qw = q0 + w * WQ;
  const int len = win_length(p, b), d = p.d;
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* vb = (const E*)p.v.ptr + b * p.v.sb + (h / p.rep) * p.v.sh;
  const int64_t row0 = ((int64_t)b * p.H + h) * p.T;

  f8 qf[NQ][KB], dof[NQ][KB];
  floatx4 acc[NQ][DB];
  float lse[NQ], del[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int t = qw + 16 * n + l16;
    const bool on = t < len;
    const E* q = (const E*)p.q.ptr + b * p.q.sb + h * p.q.sh + (int64_t)t * p.q.st;
    const E* dout = (const E*)p.dout.ptr + b * p.dout.sb + h * p.dout.sh + (int64_t)t * p.dout.st;
    const E* out = (const E*)p.out.ptr + b * p.out.sb + h * p.out.sh + (int64_t)t * p.out.st;
    const E* low = (const E*)p.low.ptr + b * p.low.sb + h * p.low.sh + (int64_t)t * p.low.st;
    float s = 0.f;
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) {
      qf[n][kk] = win_row8(q, 32 * kk + 8 * g, d, on);
      dof[n][kk] = win_row8(dout, 32 * kk + 8 * g, d, on);
      const f8 o = win_row8(out, 32 * kk + 8 * g, d, on), r = win_row8(low, 32 * kk + 8 * g, d, on && p.low.ptr);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(tof(o[e]) + tof(r[e]), tof(dof[n][kk][e]), s);
    }
    del[n] = sum_g(s);
    lse[n] = on ? p.lse[row0 + t] : INFINITY;
    if (g == 0 && t < p.T) p.delta[row0 + t] = del[n];
  }

  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[n][db] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (q0 >= len) return;
    const WinTiles tiles(q0, min(q0 + QT, len), p.window, p.sinks);
    WinTile<E, D> kr, vr;
    kr.init(p.k.st, d, tid);
    vr.init(p.v.st, d, tid);
    kr.fetch(kb, p.k.st, tiles.at(0), len);
    vr.fetch(vb, p.v.st, tiles.at(0), len);
    for (int it = 0; it < tiles.n; ++it) {
      const int k0 = tiles.at(it);
      if (it) __syncthreads();  // the last tile is read
      kr.store(kt);
      vr.store(vt);
      if (it + 1 < tiles.n) {
        kr.fetch(kb, p.k.st, tiles.at(it + 1), len);
        vr.fetch(vb, p.v.st, tiles.at(it + 1), len);
      }
      __syncthreads();
      const int cut = win_cut(qw, qw + WQ - 1, k0, p.window, p.sinks);  // wave-uniform
      if (cut == kWinNone) continue;
      floatx4 s[NQ][4];
#pragma unroll
      for (int kf = 0; kf < 4; ++kf) {
        floatx4 dp[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][kf] = dp[n] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) {
          const f8 a = IO::ld8(kt + (kf * 16 + l16) * P + 32 * kk + 8 * g);
          const f8 c = IO::ld8(vt + (kf * 16 + l16) * P + 32 * kk + 8 * g);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            s[n][kf] = mma32(a, qf[n][kk], s[n][kf]);
            dp[n] = mma32(c, dof[n][kk], dp[n]);
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[n][kf][i] = __builtin_amdgcn_exp2f(fmaf(s[n][kf][i], p.scale2, -lse[n])) * (dp[n][i] - del[n]);
      }
      if (cut != kWinWhole) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          win_mask(cut, qw + 16 * n + l16, k0, g, p.window, p.sinks, [&](int kf, int e, bool hidden) {
            s[n][kf][e] = hidden ? 0.f : s[n][kf][e];
          });
      }
      if constexpr (CAREFUL) {
        for (int gg = 0; gg < 4; ++gg)
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int kf = 0; kf < 4; ++kf)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float x = __shfl(s[n][kf][i], gg * 16 + l16, 64);
                const int key = kf * 16 + 4 * gg + i;
                if (!win_hidden(qw + 16 * n + l16, k0 + key, p.window, p.sinks))
#pragma unroll
                  for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                      acc[n][db][e] = fmaf(x, tof(kt[key * P + db * 16 + 4 * g + e]), acc[n][db][e]);
              }
        continue;
      }
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        f8 ds[NQ], rest[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          ds[n] = IO::from_acc(s[n][2 * kp], s[n][2 * kp + 1]);
          if constexpr (sizeof(E) == 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) rest[n][e] = (E)(s[n][2 * kp + (e >> 2)][e & 3] - tof(ds[n][e]));
          }
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const f8 a = TF::get(kt, P, db * 16, kp, lane);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            acc[n][db] = mma32(a, ds[n], acc[n][db]);
            if constexpr (sizeof(E) == 2) acc[n][db] = mma32(a, rest[n], acc[n][db]);
          }
        }
      }
    }
  };
  pass(std::false_type{});
  if (__syncthreads_or(win_odd<NQ, DB>(acc))) pass(std::true_type{});
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int t = qw + 16 * n + l16;
    if (t >= p.T) continue;
    const bool on = t < len;
    E* row = (E*)p.dq.ptr + b * p.dq.sb + h * p.dq.sh + (int64_t)t * p.dq.st + 4 * g;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      if (db * 16 + 4 * g >= d) continue;
      float r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = on ? acc[n][db][i] * p.scale : 0.f;
      st4f<E>(row + db * 16, r);
    }
  }
}

// A wave owns 16 NK keys.  blockIdx.x: the owners of each batch (key heads, over the query heads that share
// them, or query heads); blockIdx.y: the key tiles over the queries of their window, then the sinks'
// tiles over the queries behind it, a stretch of chunk_tiles query tiles each.
template <typename E, int D, int NK>
__global__ __launch_bounds__(256, sizeof(E) == 2 ? (D * NK == 64 ? 4 : 2) : 1) void window_dkv_kernel(WinP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  constexpr int P = win_pitch<E, D>(), DB = D / 16, KB = D / 32, WK = 16 * NK, KT = 4 * WK;
  extern __shared__ __align__(16) unsigned char lds[];
  E* qt = (E*)lds;  // [TT * P]
  E* ot = qt + TT * P;
  float* ls = (float*)(ot + TT * P);  // [TT]
  float* dl = ls + TT;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / p.owners, own = blockIdx.x % p.owners;
  const int h0 = own * p.reps, hk = h0 / p.rep;  // the first query head, and the key head
  const int len = win_length(p, b), d = p.d;
  const bool far = (int)blockIdx.y >= p.near_tiles;
  const int item = far ? (int)blockIdx.y - p.near_tiles : (int)blockIdx.y;
  const int k0 = (far ? item % p.far_tiles : item) * KT, chunk = far ? item / p.far_tiles : 0;
  const int kw = k0 + w * WK;  // this wave's first key
  // the query tiles (64 queries) that see these keys
  int t0 = k0 / TT, t1 = (min(len, k0 + KT - 1 + p.window) + TT - 1) / TT;
  if (far) {
    t0 = (k0 + p.window) / TT + chunk * p.chunk_tiles;
    t1 = min((len + TT - 1) / TT, t0 + p.chunk_tiles);
  }
  const int per_head = k0 < len ? max(0, t1 - t0) : 0, total = per_head * p.reps;
  // a query is one of this workgroup's where its distance from the key lies in least .. least + span - 1
  const uint32_t least = far ? (uint32_t)p.window : 0u, span = far ? 0x7fffffffu - (uint32_t)p.window : (uint32_t)p.window;

  f8 kf[NK][KB], vf[NK][KB];
  floatx4 dk[NK][DB], dv[NK][DB];
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int t = kw + 16 * n + l16;
    const E* k = (const E*)p.k.ptr + b * p.k.sb + hk * p.k.sh + (int64_t)t * p.k.st;
    const E* v = (const E*)p.v.ptr + b * p.v.sb + hk * p.v.sh + (int64_t)t * p.v.st;
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) {
      kf[n][kk] = win_row8(k, 32 * kk + 8 * g, d, t < len);
      vf[n][kk] = win_row8(v, 32 * kk + 8 * g, d, t < len);
    }
  }

  auto pass = [&](auto careful) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int db = 0; db < DB; ++db) dk[n][db] = dv[n][db] = floatx4{0.f, 0.f, 0.f, 0.f};
    WinTile<E, D> qr, dr;
    qr.init(p.q.st, d, tid);
    dr.init(p.dout.st, d, tid);
    float lr = INFINITY, er = 0.f;
    int at_h = h0, at_t = t0;  // of the tile on its way
    auto fetch = [&]() {
      const int q0 = at_t * TT;
      qr.fetch((const E*)p.q.ptr + b * p.q.sb + at_h * p.q.sh, p.q.st, q0, len);
      dr.fetch((const E*)p.dout.ptr + b * p.dout.sb + at_h * p.dout.sh, p.dout.st, q0, len);
      if (tid < TT) {
        const bool on = q0 + tid < len;
        const int64_t at = ((int64_t)b * p.H + at_h) * p.T + q0 + tid;
        lr = on ? p.lse[at] : INFINITY;  // (no query: its probabilities are zero)
        er = on ? p.delta[at] : 0.f;
      }
    };
    if (total) fetch();
    for (int it = 0; it < total; ++it) {
      const int q0 = at_t * TT;
      if (it) __syncthreads();  // the last tile is read
      qr.store(qt);
      dr.store(ot);
      if (tid < TT) {
        ls[tid] = lr;
        dl[tid] = er;
      }
      if (++at_t == t0 + per_head) {
        at_t = t0;
        ++at_h;
      }
      if (it + 1 < total) fetch();
      __syncthreads();
      // wave-uniform: none of these queries sees a key here, or all of them all
      const int q1 = q0 + TT - 1, k1 = kw + WK - 1;
      if (far ? kw >= p.sinks || q1 - kw < p.window : kw > q1 || q0 - k1 >= p.window) continue;
      const bool some = far ? k1 >= p.sinks || q0 - k1 < p.window : k1 > q0 || q1 - kw >= p.window;
#pragma unroll
      for (int qp = 0; qp < 2; ++qp) {
        floatx4 s[NK][2], dp[NK][2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int qf = 2 * qp + f;
#pragma unroll
          for (int n = 0; n < NK; ++n) s[n][f] = dp[n][f] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < KB; ++kk) {
            const f8 a = IO::ld8(qt + (qf * 16 + l16) * P + 32 * kk + 8 * g);
            const f8 c = IO::ld8(ot + (qf * 16 + l16) * P + 32 * kk + 8 * g);
#pragma unroll
            for (int n = 0; n < NK; ++n) {
              s[n][f] = mma32(a, kf[n][kk], s[n][f]);
              dp[n][f] = mma32(c, vf[n][kk], dp[n][f]);
            }
          }
          const floatx4 l4 = *(const floatx4*)(ls + qf * 16 + 4 * g), d4 = *(const floatx4*)(dl + qf * 16 + 4 * g);
#pragma unroll
          for (int n = 0; n < NK; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s[n][f][i] = __builtin_amdgcn_exp2f(fmaf(s[n][f][i], p.scale2, -l4[i]));
              dp[n][f][i] -= d4[i];
            }
            if (some) {
              // the distance of query i from this lane's key is c + i
              const int key = kw + 16 * n + l16, c = q0 + qf * 16 + 4 * g - key;
              const uint32_t from = far && key >= p.sinks ? 0x7fffffffu : least;
#pragma unroll
              for (int i = 0; i < 4; ++i) s[n][f][i] = (uint32_t)(c + i) - from < span ? s[n][f][i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) dp[n][f][i] *= s[n][f][i];
          }
        }
        if constexpr (CAREFUL) {
#pragma unroll 1
          for (int gg = 0; gg < 4; ++gg)
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
              for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float x = __shfl(s[n][f][i], gg * 16 + l16, 64), y = __shfl(dp[n][f][i], gg * 16 + l16, 64);
                  const int row = (2 * qp + f) * 16 + 4 * gg + i, key = kw + 16 * n + l16;
                  const uint32_t from = far && key >= p.sinks ? 0x7fffffffu : least;
                  if (q0 + row < len && (uint32_t)(q0 + row - key) - from < span)
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                      for (int e = 0; e < 4; ++e) {
                        dv[n][db][e] = fmaf(x, tof(ot[row * P + db * 16 + 4 * g + e]), dv[n][db][e]);
                        dk[n][db][e] = fmaf(y, tof(qt[row * P + db * 16 + 4 * g + e]), dk[n][db][e]);
                      }
                }
          continue;
        }
        f8 pf[NK], ef[NK];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          pf[n] = IO::from_acc(s[n][0], s[n][1]);
          ef[n] = IO::from_acc(dp[n][0], dp[n][1]);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const f8 a = TF::get(ot, P, db * 16, qp, lane), c = TF::get(qt, P, db * 16, qp, lane);
#pragma unroll
          for (int n = 0; n < NK; ++n) {
            dv[n][db] = mma32(a, pf[n], dv[n][db]);
            dk[n][db] = mma32(c, ef[n], dk[n][db]);
          }
        }
      }
    }
  };
  pass(std::false_type{});
  const bool odd = win_odd<NK, DB>(dk) | win_odd<NK, DB>(dv);
  if (__builtin_expect(__syncthreads_or(odd), 0)) pass(std::true_type{});
  const int64_t bo = (int64_t)b * p.owners + own;
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int t = kw + 16 * n + l16;
    if (t >= p.T || (far && t >= p.sinks)) continue;
    const bool on = t < len;
    const bool sink = p.chunks && t < p.sinks;
    if (sink || p.rows) {  // in parts
      float* row = (sink ? p.part + ((bo * (p.chunks + 1) + (far ? chunk + 1 : 0)) * p.sinks + t) * 2 * d
                         : p.rows + (bo * p.T + t) * 2 * d) + 4 * g;
#pragma unroll
      for (int db = 0; db < DB; ++db)
        if (db * 16 + 4 * g < d) {
          *(floatx4*)(row + db * 16) = on ? dk[n][db] : floatx4{0.f, 0.f, 0.f, 0.f};
          *(floatx4*)(row + d + db * 16) = on ? dv[n][db] : floatx4{0.f, 0.f, 0.f, 0.f};
        }
      continue;
    }
    E* krow = (E*)p.dk.ptr + b * p.dk.sb + hk * p.dk.sh + (int64_t)t * p.dk.st + 4 * g;
    E* vrow = (E*)p.dv.ptr + b * p.dv.sb + hk * p.dv.sh + (int64_t)t * p.dv.st + 4 * g;
#pragma unroll
    for (int db = 0; db < DB; ++db)
      if (db * 16 + 4 * g < d) {
        float rk[4], rv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rk[i] = on ? dk[n][db][i] * p.scale : 0.f;
          rv[i] = on ? dv[n][db][i] : 0.f;
        }
        st4f<E>(krow + db * 16, rk);
        st4f<E>(vrow + db * 16, rv);
      }
  }
}

// Gradients that stand in parts, four values a thread: the sum over the query heads that share a key head (where
// each has its own), and of a sink's row over the near queries' and the stretches', in order.
template <typename E>
__global__ __launch_bounds__(256) void window_parts_kernel(WinP p) {
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv, quads = p.d / 2;
  const int64_t at = (int64_t)blockIdx.y * 256 + threadIdx.x;
  const int t = (int)(at / quads), c = (int)(at % quads) * 4;
  if (t >= (p.rows ? p.T : p.sinks)) return;
  const int heads = p.owners / p.Hkv;
  const bool sink = p.chunks && t < p.sinks;
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < heads; ++i) {
    const int64_t bo = (int64_t)b * p.owners + hk * heads + i;
    if (!sink) {
      sum += *(const floatx4*)(p.rows + (bo * p.T + t) * 2 * p.d + c);
      continue;
    }
    const float* part = p.part + (bo * (p.chunks + 1) * p.sinks + t) * 2 * p.d + c;
#pragma unroll 4
    for (int k = 0; k <= p.chunks; ++k) sum += *(const floatx4*)(part + (int64_t)k * p.sinks * 2 * p.d);
  }
  const ts_strided& to = c < p.d ? p.dk : p.dv;
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = c < p.d ? sum[i] * p.scale : sum[i];
  st4f<E>((E*)to.ptr + b * to.sb + hk * to.sh + (int64_t)t * to.st + c % p.d, r);
}

// Keys of a workgroup of the second kernel: 128 where their sums fit twice in a SIMD's registers and workgroups
// are many (with gradients in us, 128 and 64 keys, 64-wide heads, at 128, 256, 512 and 1024 of the former: 2048
// tokens of 8 key heads 89 74, 109 105, 137 134, 221 222; 4096 of 4 131 124, 175 165, 260 258, 438 453).
static int window_keys(const WinP& p, int B, bool bf) { return bf && p.d <= 64 && !window_narrow(p, B, bf, p.Hkv) ? 128 : 64; }

struct WinSplit {
  size_t delta, rows, part;  // bytes
  size_t all() const { return delta + rows + part; }
};
// How the backward is split, and its workspace.
static WinSplit window_split(const ts_window_desc* d, WinP* p) {
  const bool bf = d->dtype == TS_BF16;
  const int keys = window_keys(*p, d->B, bf);
  p->near_tiles = (p->T + keys - 1) / keys;
  // query heads apart, where the key heads' workgroups would leave half of the CUs idle (8 on 2 heads, with
  // gradients in us, apart and together, at 32, 64, 128 and 256 of those: 64-wide 48 79, 54 114, 78 132, 108
  // 162; 128-wide 69 112, 77 154, 116 179, 175 234: the border could lie higher)
  const bool apart = p->rep > 1 && (int64_t)d->B * d->Hkv * p->near_tiles < 128;
  p->owners = apart ? d->H : d->Hkv;
  p->reps = apart ? 1 : p->rep;
  p->far_tiles = p->chunks = 0;
  const int behind = p->T - p->window;  // queries that see a sink behind their window
  if (p->sinks > 0 && behind > 0) {
    const int tiles = (behind + TT - 1) / TT + 1;
    p->far_tiles = (p->sinks + keys - 1) / keys;
    // Stretches of 16 tiles, of 4 where few workgroups are (us with gradients: one sequence of 16384 tokens of 8
    // heads on 2 in stretches of 4, 8, 16 and 32 tiles 291, 286, 308, 411; of 3000 in 1, 2, 4, 8 and 16 65, 59, 54, 58,
    // 64).  Only until every CU has several workgroups: each leaves sums of all the sinks' rows (8192
    // sinks of 32 heads of 64 in 31 stretches of 32768 queries were 4.4 GB, in one they are 0.3)
    const int64_t groups = (int64_t)d->B * p->owners * p->far_tiles, most = groups < 2048 ? 2048 / groups : 1;
    p->chunk_tiles = max(max(apart ? 4 : 16, (tiles + 63) / 64), (int)((tiles + most - 1) / most));
    p->chunks = (tiles + p->chunk_tiles - 1) / p->chunk_tiles;
  }
  WinSplit s;
  s.delta = ((size_t)d->B * d->H * d->T * 4 + 15) / 16 * 16;
  s.rows = apart ? (size_t)d->B * d->H * d->T * 2 * d->d * 4 : 0;
  s.part = p->chunks ? (size_t)d->B * p->owners * (p->chunks + 1) * p->sinks * 2 * d->d * 4 : 0;
  return s;
}

// Whether the backward takes a call: the forward that keeps what it needs asks too.
static int window_bwd_fits(const WinP& p) {
  // (a launch counts its rows of workgroups in 16 bits)
  if ((int64_t)p.near_tiles + (int64_t)p.far_tiles * p.chunks > 65535 || (int64_t)p.sinks * p.d / 2 > 65535 * 256)
    return fail(TS_ERR_NOT_IMPLEMENTED, "window attention bwd: too many tokens or sinks");
  return TS_OK;
}
int window_bwd_takes(const ts_window_desc* d, WinP p) {
  window_split(d, &p);
  return window_bwd_fits(p);
}

template <typename E, int D, int NQ, int NK>
static int window_bwd(const WinP& p, int B, hipStream_t stream) {
  const int tile = TT * win_pitch<E, D>() * (int)sizeof(E), lds = 2 * tile, ldskv = lds + 2 * TT * 4;
  hipError_t e = ensure_lds_limit((const void*)window_dq_kernel<E, D, NQ>, lds);
  if (e == hipSuccess) e = ensure_lds_limit((const void*)window_dkv_kernel<E, D, NK>, ldskv);
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention bwd: %s", hipGetErrorString(e));
  const unsigned queries = (unsigned)((p.T + 64 * NQ - 1) / (64 * NQ));
  hipLaunchKernelGGL((window_dq_kernel<E, D, NQ>), dim3((unsigned)(B * (int64_t)p.H), queries), dim3(256), lds, stream, p);
  hipLaunchKernelGGL((window_dkv_kernel<E, D, NK>),
                     dim3((unsigned)(B * (int64_t)p.owners), (unsigned)(p.near_tiles + p.far_tiles * p.chunks)),
                     dim3(256), ldskv, stream, p);
  if (p.chunks || p.rows) {
    const int64_t quads = (int64_t)(p.rows ? p.T : p.sinks) * (p.d / 2);
    hipLaunchKernelGGL((window_parts_kernel<E>), dim3((unsigned)(B * (int64_t)p.Hkv), (unsigned)((quads + 255) / 256)),
                       dim3(256), 0, stream, p);
  }
  e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention bwd: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}
template <int D>
static int window_bwd(const WinP& p, int B, bool bf, hipStream_t stream) {
  if (!bf) return window_bwd<float, D, 1, 1>(p, B, stream);
  if (window_narrow(p, B, bf, p.H)) return window_bwd<bf16, D, 1, 1>(p, B, stream);
  if constexpr (D == 64)
    if (window_keys(p, B, bf) == 128) return window_bwd<bf16, D, 2, 2>(p, B, stream);
  return window_bwd<bf16, D, 2, 1>(p, B, stream);
}

}  // namespace ts

extern "C" {

int ts_window_attention_bwd_workspace_bytes(const ts_window_desc* d, size_t* bytes) {
  ts::WinP p;
  int rc = ts::window_setup(d, nullptr, &p);
  if (rc) return rc;
  const size_t n = ts::window_split(d, &p).all();
  if ((rc = ts::window_bwd_fits(p))) return rc;
  if (bytes) *bytes = n;
  return TS_OK;
}

int ts_window_attention_bwd(const ts_window_desc* d, const ts_window_io* io, const ts_window_grads* grads,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
  ts::WinP p;
  if (!io || !grads) return ts::fail(TS_ERR_VALUE, "window attention bwd: missing tensors");
  int rc = ts::window_setup(d, io, &p);
  if (rc || d->T == 0) return rc;
  const bool bf = d->dtype == TS_BF16;
  for (const ts_strided* s : {&grads->dout, &grads->dq, &grads->dk, &grads->dv})
    if ((rc = ts::window_rows(*s, bf ? 8 : 4))) return rc;
  if (!io->lse) return ts::fail(TS_ERR_VALUE, "window attention bwd: needs the forward's lse");
  const ts::WinSplit need = ts::window_split(d, &p);
  if (!workspace || ((uintptr_t)workspace & 15u) || workspace_bytes < need.all())
    return ts::fail(TS_ERR_VALUE, "window attention bwd: workspace of %zu bytes, 16-byte aligned", need.all());
  if ((rc = ts::window_bwd_fits(p))) return rc;
  p.dout = grads->dout; p.dq = grads->dq; p.dk = grads->dk; p.dv = grads->dv;
  char* work = (char*)workspace;
  p.delta = (float*)work;
  p.rows = need.rows ? (float*)(work + need.delta) : nullptr;
  p.part = need.part ? (float*)(work + need.delta + need.rows) : nullptr;
  return d->d <= 64 ? ts::window_bwd<64>(p, d->B, bf, stream) : ts::window_bwd<128>(p, d->B, bf, stream);
}

}  // extern "C"
