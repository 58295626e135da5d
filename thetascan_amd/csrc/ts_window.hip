// Windowed softmax attention with sinks, forward (gfx950).
//
//   out[b, h, i] = sum_j softmax_j(scale q_i . k_j) v_j  over j <= i with i - j < window or j < sinks
//
// bf16 or fp32 [B,H,T,d] queries against [B,Hkv,T,d] keys and values (head h reads head
// h / (H / Hkv)), d to 128, each sequence to its own length.  A workgroup owns 128 (or 64) queries
// of a head, a wave 32 (16) of them, and walks the key tiles that they see (those of the sinks,
// then the window's): S^T = K Q^T leaves a lane with one query's scores, so the running
// maximum and sum are per-lane scalars, and the scores are the B operand of
// O^T += V^T P^T without leaving registers.  Scores, softmax and sums are fp32; in bf16 the
// probabilities enter the second product in bf16 (2^-9 of each, as the output's own
// rounding).  A lane's sum has them unrounded.  32768 tokens of 8 heads of 64 on 4 (window 1024): 104 us,
// 640 TFLOP/s, the matrix cores busy in a quarter of the time, other vector instructions in 40 %: the
// softmax bounds it.
//
// A product of a hidden key's zero probability with a value that is not finite would be NaN:
// where an output is not finite, the workgroup goes over its tiles again and adds only what
// each query sees.

#include "ts_window.h"

#include <string.h>

namespace ts {

// A wave owns 16 NQ queries.
template <typename E, int D, int NQ>
__global__ __launch_bounds__(256, sizeof(E) == 2 ? (D == 64 ? 3 : 2) : 128 / D) void window_fwd_kernel(WinP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  constexpr int P = win_pitch<E, D>(), DB = D / 16, KB = D / 32, WQ = 16 * NQ, QT = 4 * WQ;
  extern __shared__ __align__(16) unsigned char lds[];
  E* ks = (E*)lds;  // [2][TT * P]
  E* vs = ks + 2 * TT * P;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * QT, qw = q0 + w * WQ;
  const int len = win_length(p, b), d = p.d;
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* vb = (const E*)p.v.ptr + b * p.v.sb + (h / p.rep) * p.v.sh;
  E* ob = (E*)p.out.ptr + b * p.out.sb + h * p.out.sh;
  E* rb = p.low.ptr ? (E*)p.low.ptr + b * p.low.sb + h * p.low.sh : nullptr;
  float* lse = p.lse ? p.lse + ((int64_t)b * p.H + h) * p.T : nullptr;

  f8 qf[NQ][KB];
  floatx4 o[NQ][DB];
  float mx[NQ], sum[NQ];  // the scores' reference, and this lane's keys' sum from it
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int t = qw + 16 * n + l16;
    const E* row = (const E*)p.q.ptr + b * p.q.sb + h * p.q.sh + (int64_t)t * p.q.st;
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) qf[n][kk] = win_row8(row, 32 * kk + 8 * g, d, t < len);
  }
  // The reference is the highest score so far or up to 2^8 below it: terms to 2^8 lose nothing, and the
  // sums are seldom scaled.
  // (the least scales have no such slack in fp32: 1e38 of their scores is less than 2^8)
  const float slack = fminf(8.f / p.scale2, 1e38f);

  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      mx[n] = -INFINITY;
      sum[n] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[n][db] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    if (q0 >= len) return;
    const WinTiles tiles(q0, min(q0 + QT, len), p.window, p.sinks);
    WinTile<E, D> kr, vr;
    kr.init(p.k.st, d, tid);
    vr.init(p.v.st, d, tid);
    kr.fetch(kb, p.k.st, tiles.at(0), len);
    vr.fetch(vb, p.v.st, tiles.at(0), len);
    for (int it = 0; it < tiles.n; ++it) {
      const int k0 = tiles.at(it), buf = it & 1;
      E *kt = ks + buf * TT * P, *vt = vs + buf * TT * P;
      kr.store(kt);
      vr.store(vt);
      if (it + 1 < tiles.n) {
        kr.fetch(kb, p.k.st, tiles.at(it + 1), len);
        vr.fetch(vb, p.v.st, tiles.at(it + 1), len);
      }
      // this tile is staged; the other buffer, read in the last round, is free
      // once every wave has passed here, and is written only after it
      __syncthreads();
      const int cut = win_cut(qw, qw + WQ - 1, k0, p.window, p.sinks);  // wave-uniform
      if (cut == kWinNone) continue;
      floatx4 s[NQ][4];
#pragma unroll
      for (int kf = 0; kf < 4; ++kf) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][kf] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) {
          const f8 a = IO::ld8(kt + (kf * 16 + l16) * P + 32 * kk + 8 * g);
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][kf] = mma32(a, qf[n][kk], s[n][kf]);
        }
      }
      if (cut != kWinWhole) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          win_mask(cut, qw + 16 * n + l16, k0, g, p.window, p.sinks, [&](int kf, int e, bool hidden) {
            s[n][kf][e] = hidden ? -INFINITY : s[n][kf][e];
          });
      }
      float m[NQ];
      bool higher = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        m[n] = s[n][0][0];
#pragma unroll
        for (int kf = 0; kf < 4; ++kf)
#pragma unroll
          for (int i = 0; i < 4; ++i) m[n] = fmaxf(m[n], s[n][kf][i]);
        higher |= m[n] > mx[n] + slack;
      }
      if (__any(higher)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const float top = fmaxf(mx[n], max_g(m[n]));
          // (a query that has seen nothing yet has nothing to scale)
          const float fac = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mx[n] - top) * p.scale2);
          mx[n] = top;
          sum[n] *= fac;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][db][i] *= fac;
        }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float c = mx[n] == -INFINITY ? 0.f : mx[n] * p.scale2;
#pragma unroll
        for (int kf = 0; kf < 4; ++kf)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[n][kf][i] = __builtin_amdgcn_exp2f(fmaf(s[n][kf][i], p.scale2, -c));
            sum[n] += s[n][kf][i];
          }
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
                      o[n][db][e] = fmaf(x, tof(vt[key * P + db * 16 + 4 * g + e]), o[n][db][e]);
              }
      } else {
#pragma unroll
        for (int kp = 0; kp < 2; ++kp) {
          f8 pf[NQ];
#pragma unroll
          for (int n = 0; n < NQ; ++n) pf[n] = IO::from_acc(s[n][2 * kp], s[n][2 * kp + 1]);
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const f8 a = TF::get(vt, P, db * 16, kp, lane);
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[n][db] = mma32(a, pf[n], o[n][db]);
          }
        }
      }
    }
  };
  pass(std::false_type{});
  bool odd = false;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    sum[n] = sum_g(sum[n]);
    // (a sum of magnitudes is finite where all are, or where none is near the border of its type)
    float all = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) all += fabsf(o[n][db][i]);
    odd |= !(all < INFINITY);
  }
  if (__syncthreads_or(odd)) {
    pass(std::true_type{});
#pragma unroll
    for (int n = 0; n < NQ; ++n) sum[n] = sum_g(sum[n]);
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int t = qw + 16 * n + l16;
    if (t >= p.T) continue;
    const bool on = t < len;
    const float inv = on ? 1.0f / sum[n] : 0.f;
    if (lse && g == 0) lse[t] = on ? fmaf(mx[n], p.scale2, __log2f(sum[n])) : INFINITY;
    E* row = ob + (int64_t)t * p.out.st + 4 * g;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      if (db * 16 + 4 * g >= d) continue;
      float r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = on ? o[n][db][i] * inv : 0.f;
      st4f<E>(row + db * 16, r);
      if (rb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] -= tof(cvt<E>(r[i]));
        st4f<E>(rb + (int64_t)t * p.low.st + 4 * g + db * 16, r);
      }
    }
  }
}

}  // namespace ts

namespace ts {

// Rows (feature axis contiguous) of 16-byte alignment at every stride, 64 of them within 2 GiB.
int window_rows(const ts_strided& s, int vec) {
  if (!s.ptr || ((uintptr_t)s.ptr & 15u) || s.sb % vec || s.sh % vec || s.st % vec || s.st < 0)
    return fail(TS_ERR_VALUE, "window attention: rows must be 16-byte aligned");
  if (s.st >= (int64_t)1 << 23) return fail(TS_ERR_NOT_IMPLEMENTED, "window attention: rows too far apart");
  return TS_OK;
}

// The kernels' parameters of a call; without io, of its sizes.
int window_setup(const ts_window_desc* d, const ts_window_io* io, WinP* p) {
  if (!d || d->B < 1 || d->H < 1 || d->Hkv < 1 || d->H % d->Hkv || d->T < 0 || d->d < 1 || d->window < 1 ||
      d->sinks < 0 || !(d->scale >= 1.17549435e-38f && d->scale * 1.44269504088896340736f < INFINITY))
    return fail(TS_ERR_VALUE, "window attention: bad shape, window, sinks or scale");
  if (d->dtype != TS_BF16 && d->dtype != TS_F32)
    return fail(TS_ERR_NOT_IMPLEMENTED, "window attention: bf16 or fp32 only");
  const int vec = d->dtype == TS_BF16 ? 8 : 4;
  if (d->d > 128 || d->d % vec)
    return fail(TS_ERR_NOT_IMPLEMENTED, "window attention: heads of at most 128, in 16-byte vectors, got %d", d->d);
  // (a launch counts its threads in 32 bits, its rows of workgroups in 16; the smallest have 64 queries)
  if (d->T > 65535 * 64 || (int64_t)d->B * d->H * 256 >= (int64_t)1 << 32)
    return fail(TS_ERR_NOT_IMPLEMENTED, "window attention: grid too large");
  memset(p, 0, sizeof(*p));
  p->H = d->H; p->Hkv = d->Hkv; p->rep = d->H / d->Hkv; p->T = d->T; p->d = d->d;
  // (a window past the sequence is the sequence: no sum of a position and a window leaves 32 bits)
  p->window = d->window < d->T ? d->window : (d->T > 0 ? d->T : 1);
  p->sinks = d->sinks < d->T ? d->sinks : d->T;
  if (p->window >= d->T) p->sinks = 0;
  p->scale = d->scale;
  p->scale2 = d->scale * 1.44269504088896340736f;
  if (!io || d->T == 0) return TS_OK;
  for (const ts_strided* s : {&io->q, &io->k, &io->v, &io->out, io->low.ptr ? &io->low : &io->out})
    if (const int rc = window_rows(*s, vec)) return rc;
  p->q = io->q; p->k = io->k; p->v = io->v; p->out = io->out;
  p->lengths = io->lengths; p->lse = io->lse; p->low = io->low;
  return TS_OK;
}

// Whether waves own 16 rows instead of 32: fp32, whose products take 16 times the time of bf16's, and
// calls of few workgroups.  bf16 in us, 16 and 32, at 128, 256, 384, 512 and 1024 workgroups of 128 queries
// (window 1024): forward of 64-wide heads 19 27, 23 27, 26 28, 30 30, 50 48; of 128-wide 26 37, 34 39, 50 42,
// 55 45, 100 77; with gradients of 64-wide 93 110, 113 123, 123 131, 160 161, 221 219, of 128-wide 133 159, 169
// 179, 197 192, 231 220, 426 392.
bool window_narrow(const WinP& p, int B, bool bf, int heads) {
  return !bf || (int64_t)B * heads * ((p.T + 127) / 128) < 256;
}

int window_bwd_takes(const ts_window_desc* d, WinP p);

template <typename E, int D, int NQ>
static int window_fwd(const WinP& p, int B, hipStream_t stream) {
  const int lds = 4 * TT * win_pitch<E, D>() * (int)sizeof(E);
  hipError_t e = ensure_lds_limit((const void*)window_fwd_kernel<E, D, NQ>, lds);
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention: %s", hipGetErrorString(e));
  const dim3 grid((unsigned)(B * (int64_t)p.H), (unsigned)((p.T + 64 * NQ - 1) / (64 * NQ)));
  hipLaunchKernelGGL((window_fwd_kernel<E, D, NQ>), grid, dim3(256), lds, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}
template <int D>
static int window_fwd(const WinP& p, int B, bool bf, hipStream_t stream) {
  if (!bf) return window_fwd<float, D, 1>(p, B, stream);
  return window_narrow(p, B, bf, p.H) ? window_fwd<bf16, D, 1>(p, B, stream) : window_fwd<bf16, D, 2>(p, B, stream);
}

}  // namespace ts

extern "C" {

int ts_window_attention_fwd(const ts_window_desc* d, const ts_window_io* io, hipStream_t stream) {
  ts::WinP p;
  if (!io) return ts::fail(TS_ERR_VALUE, "window attention: missing tensors");
  int rc = ts::window_setup(d, io, &p);
  if (rc || d->T == 0) return rc;
  // (kept for a backward: what that refuses is refused here)
  if (io->lse && (rc = ts::window_bwd_takes(d, p))) return rc;
  const bool bf = d->dtype == TS_BF16;
  return d->d <= 64 ? ts::window_fwd<64>(p, d->B, bf, stream) : ts::window_fwd<128>(p, d->B, bf, stream);
}

}  // extern "C"
