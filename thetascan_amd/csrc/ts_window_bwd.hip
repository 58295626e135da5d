// Windowed softmax attention with sinks, backward (gfx950).
//
// With P = 2^(scale2 q k - lse), dP = dout v^T and D = rowsum(dout out):
//   dS = P (dP - D),  dv = P^T dout,  dk = scale dS^T q,  dq = scale dS k
//
// The scores are formed again, from q, k and the forward's lse.  Two kernels: one owns
// queries (dq, and D, which the other reads), one owns keys (dk and dv, over the query heads
// that share them, so that their sums have a fixed order).  Each wave keeps the rows that it
// owns as MFMA operands and accumulates in fp32; what it walks over is staged in LDS once
// for both of its uses, by rows and by columns.  In bf16, P and dS enter their products in
// bf16 (2^-9 of each).
//
// A sink is seen by every query behind its window: those pairs go to workgroups of their
// own, a stretch of queries each, which leave sums of the sinks' rows in fp32; a third kernel
// adds them in order.

#include "ts_window.h"

#include <string.h>

namespace ts {

int window_setup(const ts_window_desc* d, const ts_window_io* io, WinP* p);

template <typename E, int D>
__global__ __launch_bounds__(256) void window_dq_kernel(WinP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  constexpr int P = win_pitch<E, D>(), DB = D / 16, KB = D / 32;
  extern __shared__ __align__(16) unsigned char lds[];
  E* kt = (E*)lds;  // [TT * P]
  E* vt = kt + TT * P;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * kWinQ, qw = q0 + w * 32;
  const int len = win_length(p, b), d = p.d;
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* vb = (const E*)p.v.ptr + b * p.v.sb + (h / p.rep) * p.v.sh;
  const int64_t row0 = ((int64_t)b * p.H + h) * p.T;

  f8 qf[2][KB], dof[2][KB];
  floatx4 acc[2][DB];
  float lse[2], del[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = qw + 16 * n + l16;
    const bool on = t < len;
    const E* q = (const E*)p.q.ptr + b * p.q.sb + h * p.q.sh + (int64_t)t * p.q.st;
    const E* dout = (const E*)p.dout.ptr + b * p.dout.sb + h * p.dout.sh + (int64_t)t * p.dout.st;
    const E* out = (const E*)p.out.ptr + b * p.out.sb + h * p.out.sh + (int64_t)t * p.out.st;
    float s = 0.f;
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) {
      qf[n][kk] = win_row8(q, 32 * kk + 8 * g, d, on);
      dof[n][kk] = win_row8(dout, 32 * kk + 8 * g, d, on);
      const f8 o = win_row8(out, 32 * kk + 8 * g, d, on);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(tof(o[e]), tof(dof[n][kk][e]), s);
    }
    del[n] = sum_g(s);
    lse[n] = on ? p.lse[row0 + t] : INFINITY;
    if (g == 0 && t < p.T) p.delta[row0 + t] = del[n];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[n][db] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  if (q0 < len) {
    const WinTiles tiles(q0, min(q0 + kWinQ, len), p.window, p.sinks);
    WinTile<E, D> kr, vr;
    kr.fetch(kb, p.k.st, tiles.at(0), len, d, tid);
    vr.fetch(vb, p.v.st, tiles.at(0), len, d, tid);
    for (int it = 0; it < tiles.n; ++it) {
      const int k0 = tiles.at(it);
      if (it) __syncthreads();  // the last tile is read
      kr.store(kt, tid);
      vr.store(vt, tid);
      if (it + 1 < tiles.n) {
        kr.fetch(kb, p.k.st, tiles.at(it + 1), len, d, tid);
        vr.fetch(vb, p.v.st, tiles.at(it + 1), len, d, tid);
      }
      __syncthreads();
      if (k0 > qw + 31 || (qw - (k0 + TT - 1) >= p.window && k0 >= p.sinks)) continue;
      const bool some = k0 + TT - 1 > qw || (qw + 31 - k0 >= p.window && k0 + TT > p.sinks);
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        floatx4 s[2][2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int kf = 2 * kp + f;
          floatx4 dp[2];
          s[0][f] = s[1][f] = dp[0] = dp[1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < KB; ++kk) {
            const f8 a = IO::ld8(kt + (kf * 16 + l16) * P + 32 * kk + 8 * g);
            const f8 c = IO::ld8(vt + (kf * 16 + l16) * P + 32 * kk + 8 * g);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              s[n][f] = mma32(a, qf[n][kk], s[n][f]);
              dp[n] = mma32(c, dof[n][kk], dp[n]);
            }
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float x = __builtin_amdgcn_exp2f(fmaf(s[n][f][i], p.scale2, -lse[n])) * (dp[n][i] - del[n]);
              if (some && win_hidden(qw + 16 * n + l16, k0 + kf * 16 + 4 * g + i, p.window, p.sinks)) x = 0.f;
              s[n][f][i] = x;
            }
        }
        const f8 d0 = IO::from_acc(s[0][0], s[0][1]), d1 = IO::from_acc(s[1][0], s[1][1]);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const f8 a = TF::get(kt, P, db * 16, kp, lane);
          acc[0][db] = mma32(a, d0, acc[0][db]);
          acc[1][db] = mma32(a, d1, acc[1][db]);
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = qw + 16 * n + l16;
    if (t >= p.T) continue;
    const float c = t < len ? p.scale : 0.f;
    E* row = (E*)p.dq.ptr + b * p.dq.sb + h * p.dq.sh + (int64_t)t * p.dq.st + 4 * g;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const float r[4] = {acc[n][db][0] * c, acc[n][db][1] * c, acc[n][db][2] * c, acc[n][db][3] * c};
      if (db * 16 + 4 * g < d) st4f<E>(row + db * 16, r);
    }
  }
}

// blockIdx.y: the key tiles (128 keys) over the queries of their window, then the sinks' tiles
// over the queries behind it, a stretch of chunk_tiles query tiles each.
template <typename E, int D>
__global__ __launch_bounds__(256) void window_dkv_kernel(WinP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  constexpr int P = win_pitch<E, D>(), DB = D / 16, KB = D / 32;
  extern __shared__ __align__(16) unsigned char lds[];
  E* qt = (E*)lds;  // [TT * P]
  E* ot = qt + TT * P;
  float* ls = (float*)(ot + TT * P);  // [TT]
  float* dl = ls + TT;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv;
  const int len = win_length(p, b), d = p.d;
  const bool far = (int)blockIdx.y >= p.near_tiles;
  const int item = far ? (int)blockIdx.y - p.near_tiles : (int)blockIdx.y;
  const int k0 = (far ? item % p.far_tiles : item) * kWinQ, chunk = far ? item / p.far_tiles : 0;
  const int kw = k0 + w * 32;  // this wave's first key
  // the query tiles (64 queries) that see these keys
  int t0 = k0 / TT, t1 = (min(len, k0 + kWinQ - 1 + p.window) + TT - 1) / TT;
  if (far) {
    t0 = (k0 + p.window) / TT + chunk * p.chunk_tiles;
    t1 = min((len + TT - 1) / TT, t0 + p.chunk_tiles);
  }
  const int per_head = k0 < len ? max(0, t1 - t0) : 0, total = per_head * p.rep;

  f8 kf[2][KB], vf[2][KB];
  floatx4 dk[2][DB], dv[2][DB];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = kw + 16 * n + l16;
    const E* k = (const E*)p.k.ptr + b * p.k.sb + hk * p.k.sh + (int64_t)t * p.k.st;
    const E* v = (const E*)p.v.ptr + b * p.v.sb + hk * p.v.sh + (int64_t)t * p.v.st;
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) {
      kf[n][kk] = win_row8(k, 32 * kk + 8 * g, d, t < len);
      vf[n][kk] = win_row8(v, 32 * kk + 8 * g, d, t < len);
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[n][db] = dv[n][db] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  WinTile<E, D> qr, dr;
  float lr = INFINITY, er = 0.f;
  auto fetch = [&](int it) {
    const int h = hk * p.rep + it / per_head, q0 = (t0 + it % per_head) * TT;
    qr.fetch((const E*)p.q.ptr + b * p.q.sb + h * p.q.sh, p.q.st, q0, len, d, tid);
    dr.fetch((const E*)p.dout.ptr + b * p.dout.sb + h * p.dout.sh, p.dout.st, q0, len, d, tid);
    if (tid < TT) {
      const bool on = q0 + tid < len;
      const int64_t at = ((int64_t)b * p.H + h) * p.T + q0 + tid;
      lr = on ? p.lse[at] : INFINITY;  // (no query: its probabilities are zero)
      er = on ? p.delta[at] : 0.f;
    }
  };
  if (total) fetch(0);
  for (int it = 0; it < total; ++it) {
    const int q0 = (t0 + it % per_head) * TT;
    if (it) __syncthreads();  // the last tile is read
    qr.store(qt, tid);
    dr.store(ot, tid);
    if (tid < TT) {
      ls[tid] = lr;
      dl[tid] = er;
    }
    if (it + 1 < total) fetch(it + 1);
    __syncthreads();
    // wave-uniform: none of these queries sees a key here, or all of them all
    if (far ? kw >= p.sinks || q0 + TT - 1 - kw < p.window : kw > q0 + TT - 1 || q0 - (kw + 31) >= p.window) continue;
    const bool some = far ? kw + 31 >= p.sinks || q0 - (kw + 31) < p.window
                          : kw + 31 > q0 || q0 + TT - 1 - kw >= p.window;
#pragma unroll
    for (int qp = 0; qp < 2; ++qp) {
      floatx4 s[2][2], dp[2][2];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int qf = 2 * qp + f;
#pragma unroll
        for (int n = 0; n < 2; ++n) s[n][f] = dp[n][f] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) {
          const f8 a = IO::ld8(qt + (qf * 16 + l16) * P + 32 * kk + 8 * g);
          const f8 c = IO::ld8(ot + (qf * 16 + l16) * P + 32 * kk + 8 * g);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            s[n][f] = mma32(a, kf[n][kk], s[n][f]);
            dp[n][f] = mma32(c, vf[n][kk], dp[n][f]);
          }
        }
        const floatx4 l4 = *(const floatx4*)(ls + qf * 16 + 4 * g), d4 = *(const floatx4*)(dl + qf * 16 + 4 * g);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = __builtin_amdgcn_exp2f(fmaf(s[n][f][i], p.scale2, -l4[i]));
            if (some) {
              const int q = q0 + qf * 16 + 4 * g + i, key = kw + 16 * n + l16;
              if (far ? key >= p.sinks || q - key < p.window : key > q || q - key >= p.window) x = 0.f;
            }
            s[n][f][i] = x;
            dp[n][f][i] = x * (dp[n][f][i] - d4[i]);
          }
      }
      const f8 p0 = IO::from_acc(s[0][0], s[0][1]), p1 = IO::from_acc(s[1][0], s[1][1]);
      const f8 e0 = IO::from_acc(dp[0][0], dp[0][1]), e1 = IO::from_acc(dp[1][0], dp[1][1]);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const f8 a = TF::get(ot, P, db * 16, qp, lane), c = TF::get(qt, P, db * 16, qp, lane);
        dv[0][db] = mma32(a, p0, dv[0][db]);
        dv[1][db] = mma32(a, p1, dv[1][db]);
        dk[0][db] = mma32(c, e0, dk[0][db]);
        dk[1][db] = mma32(c, e1, dk[1][db]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = kw + 16 * n + l16;
    if (t >= p.T || (far && t >= p.sinks)) continue;
    const bool on = t < len;
    if (p.chunks && t < p.sinks) {
      const int64_t slot = ((int64_t)b * p.Hkv + hk) * (p.chunks + 1) + (far ? chunk + 1 : 0);
      float* row = p.part + (slot * p.sinks + t) * 2 * d + 4 * g;
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

// The sinks' gradients: the near queries' sums, then the stretches' in order.
template <typename E>
__global__ __launch_bounds__(256) void window_sinks_kernel(WinP p) {
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv;
  const int per = p.sinks * 2 * p.d;  // (the host checks its size)
  const int at = blockIdx.y * 256 + threadIdx.x;
  if (at >= per) return;
  const float* part = p.part + (int64_t)blockIdx.x * (p.chunks + 1) * per + at;
  float sum = 0.f;
  for (int c = 0; c <= p.chunks; ++c) sum += part[(int64_t)c * per];
  const int t = at / (2 * p.d), col = at % (2 * p.d);
  if (col < p.d)
    ((E*)p.dk.ptr)[b * p.dk.sb + hk * p.dk.sh + (int64_t)t * p.dk.st + col] = cvt<E>(sum * p.scale);
  else
    ((E*)p.dv.ptr)[b * p.dv.sb + hk * p.dv.sh + (int64_t)t * p.dv.st + col - p.d] = cvt<E>(sum);
}

// How the backward is split, and its workspace: delta, then the sinks' sums.
static size_t window_split(const ts_window_desc* d, WinP* p) {
  p->near_tiles = (p->T + kWinQ - 1) / kWinQ;
  p->far_tiles = p->chunks = 0;
  const int behind = p->T - p->window;  // queries that see a sink behind their window
  if (p->sinks > 0 && behind > 0) {
    const int tiles = (behind + TT - 1) / TT + 1;
    p->far_tiles = (p->sinks + kWinQ - 1) / kWinQ;
    p->chunk_tiles = max(16, (tiles + 63) / 64);
    p->chunks = (tiles + p->chunk_tiles - 1) / p->chunk_tiles;
  }
  const size_t delta = ((size_t)d->B * d->H * d->T * 4 + 15) / 16 * 16;
  return delta + (p->chunks ? (size_t)d->B * d->Hkv * (p->chunks + 1) * p->sinks * 2 * d->d * 4 : 0);
}

static bool grad_rows(const ts_strided& s, int vec) {
  return s.ptr && ((uintptr_t)s.ptr & 15u) == 0 && s.sb % vec == 0 && s.sh % vec == 0 && s.st % vec == 0;
}

template <typename E, int D>
static int window_bwd(const WinP& p, int B, hipStream_t stream) {
  const int tile = TT * win_pitch<E, D>() * (int)sizeof(E), lds = 2 * tile, ldskv = lds + 2 * TT * 4;
  hipError_t e = ensure_lds_limit((const void*)window_dq_kernel<E, D>, lds);
  if (e == hipSuccess) e = ensure_lds_limit((const void*)window_dkv_kernel<E, D>, ldskv);
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention bwd: %s", hipGetErrorString(e));
  hipLaunchKernelGGL((window_dq_kernel<E, D>), dim3((unsigned)(B * (int64_t)p.H), (unsigned)p.near_tiles), dim3(256), lds,
                     stream, p);
  hipLaunchKernelGGL((window_dkv_kernel<E, D>),
                     dim3((unsigned)(B * (int64_t)p.Hkv), (unsigned)(p.near_tiles + p.far_tiles * p.chunks)), dim3(256),
                     ldskv, stream, p);
  if (p.chunks)
    hipLaunchKernelGGL((window_sinks_kernel<E>),
                       dim3((unsigned)(B * (int64_t)p.Hkv), (unsigned)((p.sinks * 2 * p.d + 255) / 256)), dim3(256), 0,
                       stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window attention bwd: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}

}  // namespace ts

extern "C" {

int ts_window_attention_bwd_workspace_bytes(const ts_window_desc* d, size_t* bytes) {
  ts::WinP p;
  const int rc = ts::window_setup(d, nullptr, &p);
  if (rc) return rc;
  const size_t n = ts::window_split(d, &p);
  if (bytes) *bytes = n;
  return TS_OK;
}

int ts_window_attention_bwd(const ts_window_desc* d, const ts_window_io* io, const ts_window_grads* grads,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
  ts::WinP p;
  if (!io || !grads) return ts::fail(TS_ERR_VALUE, "window attention bwd: missing tensors");
  const int rc = ts::window_setup(d, io, &p);
  if (rc || d->T == 0) return rc;
  const int vec = d->dtype == TS_BF16 ? 8 : 4;
  for (const ts_strided* s : {&grads->dout, &grads->dq, &grads->dk, &grads->dv})
    if (!ts::grad_rows(*s, vec)) return ts::fail(TS_ERR_VALUE, "window attention bwd: rows must be 16-byte aligned");
  if (!io->lse) return ts::fail(TS_ERR_VALUE, "window attention bwd: needs the forward's lse");
  const size_t need = ts::window_split(d, &p);
  if (!workspace || ((uintptr_t)workspace & 15u) || workspace_bytes < need)
    return ts::fail(TS_ERR_VALUE, "window attention bwd: workspace of %zu bytes, 16-byte aligned", need);
  if ((int64_t)p.near_tiles + (int64_t)p.far_tiles * p.chunks > 65535 || (int64_t)p.sinks * 2 * d->d > 65535 * 256)
    return ts::fail(TS_ERR_NOT_IMPLEMENTED, "window attention bwd: too many sinks");
  p.dout = grads->dout; p.dq = grads->dq; p.dk = grads->dk; p.dv = grads->dv;
  p.delta = (float*)workspace;
  p.part = (float*)((char*)workspace + ((size_t)d->B * d->H * d->T * 4 + 15) / 16 * 16);
  if (d->dtype == TS_BF16)
    return d->d <= 64 ? ts::window_bwd<ts::bf16, 64>(p, d->B, stream) : ts::window_bwd<ts::bf16, 128>(p, d->B, stream);
  return d->d <= 64 ? ts::window_bwd<float, 64>(p, d->B, stream) : ts::window_bwd<float, 128>(p, d->B, stream);
}

}  // extern "C"
