// Gated delta rule, token by token against a carried state (gfx950): the form
// for serving, where a call brings one token a sequence or a few.
//
//   S <- a S;  u = b (v - S^T k);  S <- S + k u^T;  o = S^T q
//
// One pass over the fp32 state: a wave owns 32 of a head's value columns (16 bytes
// of a row per lane, eight lanes a row, dk / 8 consecutive rows a lane, in
// registers), reads them once, walks the tokens and writes them once.  S^T k, S^T q
// and k.q are reduced together over the eight lanes of a column: with the decayed
// state, o = a S^T q + (k.q) u needs no second pass over the updated one.  fp32
// throughout.  A token's inputs are loaded a token ahead, as vectors, and the
// reductions are lane permutes: 0.7 us a token where heads are few (1.9 with loads
// of single elements in the token's own turn and reductions through LDS).
//
// Bound by the state's bytes where there are many heads: one token of 2048 heads of
// 128 x 128 (270 MB) 48 us, 5.6 TB/s; of 4096 of 64 x 64 (134 MB) 23 us (29 us at two
// waves a SIMD, which the compiler left it at).  Where heads are few, one memory round trip and the
// launch: 16 heads of 64 x 64 4.3 us.

#include "ts_delta.h"

namespace ts {

// What the lanes of a wave hold between them of a value: the sum over the eight row
// groups (lanes 8, 16 and 32 apart), in every lane, without LDS.
__device__ __forceinline__ float sum_rows(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, true));  // row_ror:8
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r16[0]) + __uint_as_float(r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r32[0]) + __uint_as_float(r32[1]);
}

// One token's inputs of a lane: its rows of k and q, its columns of v, the gates.
template <typename E, int ROWS>
struct StepToken {
  static constexpr int N = Vec16<E>::N, VECS = ROWS / N;
  Vec16<E> k[VECS], q[VECS];
  float v[4], be, la;
  // (rows past dk read the first ones, for clear to zero)
  __device__ __forceinline__ void fetch(const DeltaP& p, const E* kb, const E* qb, const E* vb, int64_t gb, int64_t gd,
                                        int row0, int t) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int row = row0 + i * N < p.dk ? row0 + i * N : 0;
      k[i].raw = *(const uint4*)(kb + (int64_t)t * p.k.st + row);
      q[i].raw = *(const uint4*)(qb + (int64_t)t * p.q.st + row);
    }
    ld4f<E>(vb + (int64_t)t * p.v.st, v);
    be = gate_at(p.beta, p.beta_bf16, gb + (int64_t)t * p.beta.st);
    la = p.decay.ptr ? gate_at(p.decay, p.decay_bf16, gd + (int64_t)t * p.decay.st) : 0.f;
  }
  __device__ __forceinline__ void clear(int row0, int dk) {
    if (row0 + ROWS <= dk) return;
#pragma unroll
    for (int i = 0; i < VECS; ++i)
      if (row0 + i * N >= dk) k[i].raw = q[i].raw = make_uint4(0u, 0u, 0u, 0u);
  }
};

template <typename E, int DK>
__global__ __launch_bounds__(64, DK == 64 ? 4 : 3) void delta_step_kernel(DeltaP p) {
  constexpr int ROWS = DK / 8;
  typedef StepToken<E, ROWS> Token;
  const int lane = threadIdx.x, cl = lane & 7, rl = lane >> 3;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
  const int col = (int)blockIdx.y * 32 + 4 * cl, row0 = rl * ROWS;
  const bool on = col < p.dv;
  const int len = delta_len(p, b);
  // (lanes past dv read the first columns and store nothing)
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* qb = (const E*)p.q.ptr + b * p.q.sb + (h / p.rep) * p.q.sh;
  const E* vb = (const E*)p.v.ptr + b * p.v.sb + h * p.v.sh + (on ? col : 0);
  E* ob = (E*)p.out.ptr + b * p.out.sb + h * p.out.sh + col;
  const int64_t gb = b * p.beta.sb + h * p.beta.sh, gd = b * p.decay.sb + h * p.decay.sh;
  const int64_t st0 = ((int64_t)bh * p.dk + row0) * p.dv + col;
  Token tok;
  if (len > 0) tok.fetch(p, kb, qb, vb, gb, gd, row0, 0);
  floatx4 S[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    S[j] = zero4();
    if (p.state && on && row0 + j < p.dk) S[j] = *(const floatx4*)(p.state + st0 + (int64_t)j * p.dv);
  }
  for (int t = 0; t < len; ++t) {
    Token next = tok;
    if (t + 1 < len) next.fetch(p, kb, qb, vb, gb, gd, row0, t + 1);  // uniform
    tok.clear(row0, p.dk);
    const float a = expf(tok.la);
    float ks[4] = {0.f, 0.f, 0.f, 0.f}, qs[4] = {0.f, 0.f, 0.f, 0.f}, kq = 0.f;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const float k = tof(tok.k[j / Token::N].e[j % Token::N]), q = tof(tok.q[j / Token::N].e[j % Token::N]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        S[j][i] *= a;
        ks[i] = fmaf(S[j][i], k, ks[i]);
        qs[i] = fmaf(S[j][i], q, qs[i]);
      }
      kq = fmaf(k, q, kq);
    }
    kq = sum_rows(kq);
    float u[4], out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = tok.be * (tok.v[i] - sum_rows(ks[i]));
      out[i] = fmaf(kq, u[i], sum_rows(qs[i]));
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const float k = tof(tok.k[j / Token::N].e[j % Token::N]);
#pragma unroll
      for (int i = 0; i < 4; ++i) S[j][i] = fmaf(k, u[i], S[j][i]);
    }
    if (on && rl == 0) st4f<E>(ob + (int64_t)t * p.out.st, out);
    tok = next;
  }
  if (!on) return;
  const float none[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = len + rl; t < p.T; t += 8) st4f<E>(ob + (int64_t)t * p.out.st, none);
  // (every entry is written by the lane that read it: state_out may be the state itself)
  if (p.state_out) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (row0 + j < p.dk) *(floatx4*)(p.state_out + st0 + (int64_t)j * p.dv) = S[j];
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
