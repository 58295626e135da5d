// Gated delta rule, token by token against a carried state (gfx950): the form
// for serving, where a call brings one token a sequence or a few.
//
//   S <- a S;  u = b (v - S^T k);  S <- S + k u^T;  o = S^T q
//
// One pass over the fp32 state: a wave owns 32 of a head's value columns (16
// bytes of a row per lane, eight lanes a row, every row in registers), reads
// them once, walks the tokens and writes them once.  S^T k, S^T q and k.q are
// reduced together over the eight lanes of a column: with the decayed state,
// o = a S^T q + (k.q) u needs no second pass over the updated one.  fp32
// throughout.  Bound by the state's bytes where there are many heads, by one
// memory round trip where there are few.

#include "ts_delta.h"

namespace ts {

template <typename E, int DK>
__global__ __launch_bounds__(64) void delta_step_kernel(DeltaP p) {
  constexpr int ROWS = DK / 8;
  const int lane = threadIdx.x, cl = lane & 7, rl = lane >> 3;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
  const int col = (int)blockIdx.y * 32 + 4 * cl;
  const bool on = col < p.dv;
  const int len = delta_len(p, b);
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* qb = (const E*)p.q.ptr + b * p.q.sb + (h / p.rep) * p.q.sh;
  const E* vb = (const E*)p.v.ptr + b * p.v.sb + h * p.v.sh + col;
  E* ob = (E*)p.out.ptr + b * p.out.sb + h * p.out.sh + col;
  const int64_t st0 = (int64_t)bh * p.dk * p.dv + col;
  floatx4 S[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    S[j] = zero4();
    const int row = rl + 8 * j;
    if (p.state && on && row < p.dk) S[j] = *(const floatx4*)(p.state + st0 + (int64_t)row * p.dv);
  }
  for (int t = 0; t < len; ++t) {
    float k[ROWS], q[ROWS], v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int row = rl + 8 * j;
      k[j] = row < p.dk ? tof(kb[(int64_t)t * p.k.st + row]) : 0.f;
      q[j] = row < p.dk ? tof(qb[(int64_t)t * p.q.st + row]) : 0.f;
    }
    if (on) ld4f<E>(vb + (int64_t)t * p.v.st, v);
    const float be = gate_at(p.beta, p.beta_bf16, b * p.beta.sb + h * p.beta.sh + (int64_t)t * p.beta.st);
    float a = 1.f;
    if (p.decay.ptr)
      a = expf(gate_at(p.decay, p.decay_bf16, b * p.decay.sb + h * p.decay.sh + (int64_t)t * p.decay.st));
    float ks[4] = {0.f, 0.f, 0.f, 0.f}, qs[4] = {0.f, 0.f, 0.f, 0.f}, kq = 0.f;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        S[j][i] *= a;
        ks[i] = fmaf(S[j][i], k[j], ks[i]);
        qs[i] = fmaf(S[j][i], q[j], qs[i]);
      }
      kq = fmaf(k[j], q[j], kq);
    }
#pragma unroll
    for (int o = 8; o <= 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ks[i] += __shfl_xor(ks[i], o, 64);
        qs[i] += __shfl_xor(qs[i], o, 64);
      }
      kq += __shfl_xor(kq, o, 64);
    }
    float u[4], out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = be * (v[i] - ks[i]);
      out[i] = fmaf(kq, u[i], qs[i]);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[j][i] = fmaf(k[j], u[i], S[j][i]);
    if (on && rl == 0) st4f<E>(ob + (int64_t)t * p.out.st, out);
  }
  if (!on) return;
  const float none[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = len + rl; t < p.T; t += 8) st4f<E>(ob + (int64_t)t * p.out.st, none);
  // (every entry is written by the lane that read it: state_out may be the state itself)
  if (p.state_out) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int row = rl + 8 * j;
      if (row < p.dk) *(floatx4*)(p.state_out + st0 + (int64_t)row * p.dv) = S[j];
    }
  }
}

}  // namespace ts

extern "C" int ts_delta_step(const ts_delta_desc* d, const ts_delta_io* io, hipStream_t stream) {
  using ts::fail;
  ts::DeltaP p;
  if (!io) return fail(TS_ERR_VALUE, "delta step: missing tensors");
  const int rc = ts::delta_check(d, io, &p, "delta step");
  if (rc) return rc;
  if (((uintptr_t)p.state & 15u) || ((uintptr_t)p.state_out & 15u))
    return fail(TS_ERR_VALUE, "delta step: the states must be 16-byte aligned");
  if (d->T == 0) return TS_OK;
  const dim3 grid((unsigned)(p.B * p.H), (unsigned)((p.dv + 31) / 32));
  if (d->dtype == TS_BF16) {
    if (p.dk <= 64)
      hipLaunchKernelGGL((ts::delta_step_kernel<ts::bf16, 64>), grid, dim3(64), 0, stream, p);
    else
      hipLaunchKernelGGL((ts::delta_step_kernel<ts::bf16, 128>), grid, dim3(64), 0, stream, p);
  } else {
    if (p.dk <= 64)
      hipLaunchKernelGGL((ts::delta_step_kernel<float, 64>), grid, dim3(64), 0, stream, p);
    else
      hipLaunchKernelGGL((ts::delta_step_kernel<float, 128>), grid, dim3(64), 0, stream, p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "delta step: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}
