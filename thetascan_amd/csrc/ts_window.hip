// Windowed softmax attention with sinks, forward (gfx950).
//
//   out[b, h, i] = sum_j softmax_j(scale q_i . k_j) v_j  over j <= i with i - j < window or j < sinks
//
// bf16 or fp32 [B,H,T,d] queries against [B,Hkv,T,d] keys and values (head h reads head
// h / (H / Hkv)), d to 128, each sequence to its own length.  A workgroup owns 128 queries
// of a head, a wave 32 of them, and walks the key tiles that they see (those of the sinks,
// then the window's): S^T = K Q^T leaves a lane with one query's scores, so the running
// maximum and sum are per-lane scalars, and the scores are the B operand of
// O^T += V^T P^T without leaving registers.  Scores, softmax and sums are fp32; in bf16 the
// probabilities enter the second product in bf16 (2^-9 of each, as the output's own
// rounding).  A lane's sum has them unrounded.
//
// A product of a hidden key's zero probability with a value that is not finite would be NaN:
// where an output is not finite, the workgroup goes over its tiles again and adds only what
// each query sees.

#include "ts_window.h"

#include <string.h>

namespace ts {

template <typename E, int D>
__global__ __launch_bounds__(256) void window_fwd_kernel(WinP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  constexpr int P = win_pitch<E, D>(), DB = D / 16, KB = D / 32;
  extern __shared__ __align__(16) unsigned char lds[];
  E* ks = (E*)lds;  // [2][TT * P]
  E* vs = ks + 2 * TT * P;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * kWinQ, qw = q0 + w * 32;
  const int len = win_length(p, b), d = p.d;
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* vb = (const E*)p.v.ptr + b * p.v.sb + (h / p.rep) * p.v.sh;
  E* ob = (E*)p.out.ptr + b * p.out.sb + h * p.out.sh;
  float* lse = p.lse ? p.lse + ((int64_t)b * p.H + h) * p.T : nullptr;

  f8 qf[2][KB];
  floatx4 o[2][DB];
  float mx[2], sum[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = qw + 16 * n + l16;
    const E* row = (const E*)p.q.ptr + b * p.q.sb + h * p.q.sh + (int64_t)t * p.q.st;
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) qf[n][kk] = win_row8(row, 32 * kk + 8 * g, d, t < len);
  }

  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      mx[n] = -INFINITY;
      sum[n] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[n][db] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    if (q0 >= len) return;
    const WinTiles tiles(q0, min(q0 + kWinQ, len), p.window, p.sinks);
    WinTile<E, D> kr, vr;
    kr.fetch(kb, p.k.st, tiles.at(0), len, d, tid);
    vr.fetch(vb, p.v.st, tiles.at(0), len, d, tid);
    for (int it = 0; it < tiles.n; ++it) {
      const int k0 = tiles.at(it), buf = it & 1;
      E *kt = ks + buf * TT * P, *vt = vs + buf * TT * P;
      kr.store(kt, tid);
      vr.store(vt, tid);
      if (it + 1 < tiles.n) {
        kr.fetch(kb, p.k.st, tiles.at(it + 1), len, d, tid);
        vr.fetch(vb, p.v.st, tiles.at(it + 1), len, d, tid);
      }
      // this tile is staged; the other buffer, read in the last round, is free
      // once every wave has passed here, and is written only after it
      __syncthreads();
      // wave-uniform: no query here sees a key of the tile
      if (k0 > qw + 31 || (qw - (k0 + TT - 1) >= p.window && k0 >= p.sinks)) continue;
      floatx4 s[2][4];
#pragma unroll
      for (int kf = 0; kf < 4; ++kf) {
        s[0][kf] = s[1][kf] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) {
          const f8 a = IO::ld8(kt + (kf * 16 + l16) * P + 32 * kk + 8 * g);
          s[0][kf] = mma32(a, qf[0][kk], s[0][kf]);
          s[1][kf] = mma32(a, qf[1][kk], s[1][kf]);
        }
      }
      // wave-uniform: some query here does not see some key of the tile
      if (k0 + TT - 1 > qw || (qw + 31 - k0 >= p.window && k0 + TT > p.sinks)) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int kf = 0; kf < 4; ++kf)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (win_hidden(qw + 16 * n + l16, k0 + kf * 16 + 4 * g + i, p.window, p.sinks)) s[n][kf][i] = -INFINITY;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float m = s[n][0][0];
#pragma unroll
        for (int kf = 0; kf < 4; ++kf)
#pragma unroll
          for (int i = 0; i < 4; ++i) m = fmaxf(m, s[n][kf][i]);
        m = fmaxf(mx[n], max_g(m));
        // (a query that has seen nothing yet: its terms are zero at any finite maximum)
        const float top = m == -INFINITY ? 0.f : m;
        const float fac = __builtin_amdgcn_exp2f((mx[n] - top) * p.scale2);
        const float c = top * p.scale2;
        mx[n] = m;
        float part = 0.f;
#pragma unroll
        for (int kf = 0; kf < 4; ++kf)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[n][kf][i] = __builtin_amdgcn_exp2f(fmaf(s[n][kf][i], p.scale2, -c));
            part += s[n][kf][i];
          }
        sum[n] = fmaf(sum[n], fac, part);  // this lane's keys; the lanes are added at the end
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][db][i] *= fac;
      }
      if constexpr (CAREFUL) {
        for (int gg = 0; gg < 4; ++gg)
#pragma unroll
          for (int n = 0; n < 2; ++n)
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
          const f8 p0 = IO::from_acc(s[0][2 * kp], s[0][2 * kp + 1]);
          const f8 p1 = IO::from_acc(s[1][2 * kp], s[1][2 * kp + 1]);
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const f8 a = TF::get(vt, P, db * 16, kp, lane);
            o[0][db] = mma32(a, p0, o[0][db]);
            o[1][db] = mma32(a, p1, o[1][db]);
          }
        }
      }
    }
  };
  pass(std::false_type{});
  bool odd = false;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    sum[n] = sum_g(sum[n]);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) odd |= !(fabsf(o[n][db][i]) < INFINITY);
  }
  if (__syncthreads_or(odd)) {
    pass(std::true_type{});
    sum[0] = sum_g(sum[0]);
    sum[1] = sum_g(sum[1]);
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = qw + 16 * n + l16;
    if (t >= p.T) continue;
    const bool on = t < len;
    const float inv = on ? 1.0f / sum[n] : 0.f;
    if (lse && g == 0) lse[t] = on ? fmaf(mx[n], p.scale2, __log2f(sum[n])) : INFINITY;
    E* row = ob + (int64_t)t * p.out.st + 4 * g;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const float r[4] = {on ? o[n][db][0] * inv : 0.f, on ? o[n][db][1] * inv : 0.f, on ? o[n][db][2] * inv : 0.f,
                          on ? o[n][db][3] * inv : 0.f};
      if (db * 16 + 4 * g < d) st4f<E>(row + db * 16, r);
    }
  }
}

}  // namespace ts

namespace ts {

// Rows (feature axis contiguous) of 16-byte alignment at every stride.
static bool win_rows(const ts_strided& s, int vec) {
  return s.ptr && ((uintptr_t)s.ptr & 15u) == 0 && s.sb % vec == 0 && s.sh % vec == 0 && s.st % vec == 0;
}

// The kernels' parameters of a call; `any` skips the pointers (a workspace query).
int window_setup(const ts_window_desc* d, const ts_window_io* io, WinP* p) {
  if (!d || d->B < 1 || d->H < 1 || d->Hkv < 1 || d->H % d->Hkv || d->T < 0 || d->d < 1 || d->window < 1 ||
      d->sinks < 0 || !(d->scale > 0.f && d->scale < INFINITY))
    return fail(TS_ERR_VALUE, "window attention: bad shape, window, sinks or scale");
  if (d->dtype != TS_BF16 && d->dtype != TS_F32)
    return fail(TS_ERR_NOT_IMPLEMENTED, "window attention: bf16 or fp32 only");
  const int vec = d->dtype == TS_BF16 ? 8 : 4;
  if (d->d > 128 || d->d % vec)
    return fail(TS_ERR_NOT_IMPLEMENTED, "window attention: heads of at most 128, in 16-byte vectors, got %d", d->d);
  const int64_t heads = (int64_t)d->B * d->H, tiles = ((int64_t)d->T + kWinQ - 1) / kWinQ;
  // (a launch counts its threads in 32 bits)
  if (d->T > 0x7fffffff - 2 * kWinQ || tiles > 65535 || heads * 256 >= (int64_t)1 << 32)
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
  if (!win_rows(io->q, vec) || !win_rows(io->k, vec) || !win_rows(io->v, vec) || !win_rows(io->out, vec))
    return fail(TS_ERR_VALUE, "window attention: rows must be 16-byte aligned");
  p->q = io->q; p->k = io->k; p->v = io->v; p->out = io->out;
  p->lengths = io->lengths; p->lse = io->lse;
  return TS_OK;
}

template <typename E, int D>
static int window_fwd(const WinP& p, int B, hipStream_t stream) {
  const int lds = 4 * TT * win_pitch<E, D>() * (int)sizeof(E);
  const void* fn = (const void*)window_fwd_kernel<E, D>;
  hipError_t e = ensure_lds_limit(fn, lds);
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention: %s", hipGetErrorString(e));
  const dim3 grid((unsigned)(B * (int64_t)p.H), (unsigned)((p.T + kWinQ - 1) / kWinQ));
  hipLaunchKernelGGL((window_fwd_kernel<E, D>), grid, dim3(256), lds, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}

}  // namespace ts

extern "C" {

int ts_window_attention_fwd(const ts_window_desc* d, const ts_window_io* io, hipStream_t stream) {
  ts::WinP p;
  if (!io) return ts::fail(TS_ERR_VALUE, "window attention: missing tensors");
  const int rc = ts::window_setup(d, io, &p);
  if (rc || d->T == 0) return rc;
  if (d->dtype == TS_BF16)
    return d->d <= 64 ? ts::window_fwd<ts::bf16, 64>(p, d->B, stream) : ts::window_fwd<ts::bf16, 128>(p, d->B, stream);
  return d->d <= 64 ? ts::window_fwd<float, 64>(p, d->B, stream) : ts::window_fwd<float, 128>(p, d->B, stream);
}

}  // extern "C"
