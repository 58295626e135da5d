// Gated delta rule over whole sequences, forward (gfx950); the mathematics is in
// ts_delta.h.
//
// delta_prepare: one wave a chunk, nothing shared between chunks.  K K^T and
// Q K^T on MFMA straight from global rows, the decay between every pair, and the
// inverse of the unit lower triangular I + L: the four 16 x 16 diagonal blocks by
// substitution (a lane per row), the six below them by fp32 MFMA,
// Ti_ij = -Ti_ii sum_k L_ik Ti_kj.
//
// delta_forward: the chain over the chunks.  A column of the state needs no
// other column, so a wave owns 16 value columns of one head for the whole
// sequence, its state in accumulators, and an accumulator is the next product's
// operand without leaving the registers (rows of the accumulator are the
// contraction).  Every operand that is not an input enters in three bf16 parts, which
// hold fp32's 24 bits (six products of two such operands, three with an input): the
// state, the long sum here, is off by 1.4e-7 to 2e-7 over any length, as of fp32 inputs, and
// an output is rounded once.  In two parts it is off by 4e-6, for 13 to 19 % (prompts) and
// 6 % (training) less time.
//
// Bound by the bytes where heads and tokens are many: 64 heads of 4096 tokens of 64 x 64
// (bf16, training; bytes by counters) prepare 42 us (180 MB, 4.3 TB/s), transfers 62 (145 MB),
// forward 100 (394 MB, 3.9 TB/s; four fifths of what it writes is kept for the gradients).  Where they are few,
// by the chain: 16 chunks of 64 keys 73 us, 4.5 a chunk, a workgroup a CU.  In two parts:
// workgroups of eight waves (forward of 32 heads of 2048 x 128 65 us against 56) and three waves
// a SIMD (77 against 65) were slower; P formed here again, not stored, 0.8 us more a chunk for
// 6 % less time where bytes bind.

#include "ts_delta.h"

#include <string.h>

namespace ts {

template <typename E>
__device__ __forceinline__ typename Frag<E>::f8 global8(const E* row, int c, int width, bool on) {
  constexpr int VEC = 16 / (int)sizeof(E);
  uint4 raw[8 / VEC];
#pragma unroll
  for (int i = 0; i < 8 / VEC; ++i) {
    raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (on && c + i * VEC < width) raw[i] = *(const uint4*)(row + c + i * VEC);
  }
  return __builtin_bit_cast(typename Frag<E>::f8, raw);
}

constexpr int kDiagPitch = 20;

template <typename E, int DK>
__global__ __launch_bounds__(256) void delta_prepare_kernel(DeltaP p) {
  typedef LdsIO<E> IO;
  __shared__ __align__(16) double gs[4][kChunk];
  __shared__ __align__(16) float diag[4][4 * 16 * kDiagPitch];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  const int64_t n = (int64_t)blockIdx.x * 4 + wv;
  if (n >= (int64_t)p.B * p.H * p.nc) return;
  const int c = (int)(n % p.nc), bh = (int)(n / p.nc), b = bh / p.H, h = bh % p.H;
  const int t0 = c * kChunk, len = delta_len(p, b);
  if (t0 >= len) return;
  double* G = gs[wv];
  float* dg = diag[wv];

  // log decays, their running sum, and the vectors the chain reads
  const bool seen = t0 + lane < len;
  double sum = 0.0;
  float beta = 0.f;
  if (seen) {
    beta = gate_at(p.beta, p.beta_bf16, b * p.beta.sb + h * p.beta.sh + (int64_t)(t0 + lane) * p.beta.st);
    if (p.decay.ptr) {
      const float la =
          gate_at(p.decay, p.decay_bf16, b * p.decay.sb + h * p.decay.sh + (int64_t)(t0 + lane) * p.decay.st);
      sum = la < -1000.f ? -1000.0 : (double)la;
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double below = __shfl_up(sum, o, 64);
    if (lane >= o) sum += below;
  }
  G[lane] = sum;
  float* tri_t = p.prep + n * kRecord;
  float *tri_p = tri_t + kTriElems, *vec = tri_p + kTriElems;
  const double last = __shfl(sum, 63, 64);
  const float eg = __builtin_amdgcn_exp2f((float)(sum * kLog2e));
  const float tail = __builtin_amdgcn_exp2f((float)((last - sum) * kLog2e));
  vec[lane] = seen ? eg : 0.f;
  vec[kChunk + lane] = seen ? tail : 0.f;
  vec[2 * kChunk + lane] = beta;
  if (lane == 63) vec[3 * kChunk] = eg;
  wave_lds_sync();

  // K K^T and Q K^T, the lower blocks: column t = l16 of block rt, rows i = 4g.. of block ri
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* qb = (const E*)p.q.ptr + b * p.q.sb + (h / p.rep) * p.q.sh;
  floatx4 kk[10], qk[10];
#pragma unroll
  for (int i = 0; i < 10; ++i) kk[i] = qk[i] = zero4();
#pragma unroll
  for (int s = 0; s < DK / 32; ++s) {
    typename Frag<E>::f8 kf[4], qf[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = t0 + 16 * r + l16;
      kf[r] = global8<E>(kb + (int64_t)t * p.k.st, 32 * s + 8 * g, p.dk, t < len);
      qf[r] = global8<E>(qb + (int64_t)t * p.q.st, 32 * s + 8 * g, p.dk, t < len);
    }
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
#pragma unroll
      for (int ri = 0; ri <= rt; ++ri) {
        const int at = rt * (rt + 1) / 2 + ri;
        kk[at] = mma32(kf[ri], kf[rt], kk[at]);
        qk[at] = mma32(kf[ri], qf[rt], qk[at]);
      }
  }
  // times the decay between the pair, masked: P, and L in kk
  const floatx4 z4 = zero4();
#pragma unroll
  for (int rt = 0; rt < 4; ++rt) {
    const double gt = G[16 * rt + l16];
    const float bt = __shfl(beta, 16 * rt + l16, 64);
#pragma unroll
    for (int ri = 0; ri <= rt; ++ri) {
      const int at = rt * (rt + 1) / 2 + ri;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 16 * ri + 4 * g + j, t = 16 * rt + l16;
        const float d = __builtin_amdgcn_exp2f((float)((gt - G[i]) * kLog2e));
        qk[at][j] = i <= t ? qk[at][j] * d : 0.f;
        kk[at][j] = i < t ? kk[at][j] * d * bt : 0.f;
      }
    }
#pragma unroll
    for (int s = 0; s <= rt / 2; ++s) {
      const int at = rt * (rt + 1) / 2 + 2 * s;
      put_tri(tri_p, rt, s, lane, Parts<float, 1>(qk[at], 2 * s + 1 <= rt ? qk[2 * s + 1 <= rt ? at + 1 : at] : z4));
    }
  }
  // A token that is not finite reaches none before it: the products' zeros above the diagonal
  // would not keep it out (0 NaN), so rows of L from the first such one on are left out.  What
  // is made of those rows is not finite by itself (delta_forward sees it in R).
  float off = 0.f;
#pragma unroll
  for (int at = 0; at < 10; ++at)
#pragma unroll
    for (int j = 0; j < 4; ++j) off = taint(kk[at][j], off);
  if (__any(off != off)) {
    int first = kChunk;
#pragma unroll
    for (int rt = 3; rt >= 0; --rt) {
      float row = 0.f;
#pragma unroll
      for (int ri = 0; ri <= rt; ++ri)
#pragma unroll
        for (int j = 0; j < 4; ++j) row = taint(kk[rt * (rt + 1) / 2 + ri][j], row);
      if (row != row) first = 16 * rt + l16;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
      if (16 * rt + l16 >= first)
#pragma unroll
        for (int ri = 0; ri <= rt; ++ri) kk[rt * (rt + 1) / 2 + ri] = zero4();
  }
  // diagonal blocks: block g, row l16 of it per lane.  L_gg^T in LDS, [column][row]
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) dg[(16 * r + 4 * g + j) * kDiagPitch + l16] = kk[r * (r + 1) / 2 + r][j];
  wave_lds_sync();
  float x[16];
#pragma unroll
  for (int col = 15; col >= 0; --col) {
    float lrow[16];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const floatx4 w = *(const floatx4*)(dg + (16 * g + col) * kDiagPitch + 4 * v);
#pragma unroll
      for (int j = 0; j < 4; ++j) lrow[4 * v + j] = w[j];
    }
    float acc = col == l16 ? 1.f : 0.f;
#pragma unroll
    for (int s = 15; s > col; --s) acc = fmaf(-x[s], lrow[s], acc);
    x[col] = acc;
  }
  wave_lds_sync();
#pragma unroll
  for (int v = 0; v < 4; ++v)
    *(floatx4*)(dg + (16 * g + l16) * kDiagPitch + 4 * v) = floatx4{x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]};
  wave_lds_sync();
  // ac[..]: rows in registers (the next contraction), tr[..]: columns in
  // registers (lane l16 a row), the form of the stored operands
  floatx4 ac[6], tr[10];
#pragma unroll
  for (int r = 0; r < 4; ++r) tr[r * (r + 1) / 2 + r] = *(const floatx4*)(dg + (16 * r + l16) * kDiagPitch + 4 * g);
#pragma unroll
  for (int r = 0; r < 3; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) ac[r * (r + 1) / 2 + r][j] = dg[(16 * r + 4 * g + j) * kDiagPitch + l16];
#pragma unroll
  for (int i = 1; i < 4; ++i)
#pragma unroll
    for (int j = i - 1; j >= 0; --j) {
      floatx4 y = z4;
#pragma unroll
      for (int k = j; k < i; ++k) y = mma16(kk[i * (i + 1) / 2 + k], ac[k * (k + 1) / 2 + j], y);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = -y[e];
      const floatx4 ti = tr[i * (i + 1) / 2 + i];
      tr[i * (i + 1) / 2 + j] = mma16(y, ti, z4);
      if (i < 3) ac[i * (i + 1) / 2 + j] = mma16(ti, y, z4);
    }
#pragma unroll
  for (int rt = 0; rt < 4; ++rt)
#pragma unroll
    for (int s = 0; s <= rt / 2; ++s) {
      const int at = rt * (rt + 1) / 2 + 2 * s;
      put_tri(tri_t, rt, s, lane, Parts<float, 1>(tr[at], 2 * s + 1 <= rt ? tr[2 * s + 1 <= rt ? at + 1 : at] : z4));
    }
}

// What the waves of a workgroup read of one chunk (a transfer: no queries).
template <typename E, int DK, bool TRANSFER>
struct ForwardChunk {
  static constexpr int PAD = 16 / (int)sizeof(E), PITCH = DK + PAD, VP = 64 + PAD, SET = kParts<E, 3> * kTriElems;
  E k[kChunk * PITCH], v[kChunk * VP], t[SET], p[TRANSFER ? 8 : SET], q[TRANSFER ? 8 : kChunk * PITCH];
  float vec[256];
};

// kForward: outputs.  kKeep: also U and S0 of every chunk, for the backward.
// kTransfer: what a segment of chunks makes of its entering state, S -> X S + N:
// no outputs; column blocks of X (the identity's columns, without values), then of
// N (a zero state).
enum { kForward = 0, kKeep = 1, kTransfer = 2 };

template <typename E, int DK, int MODE>
__global__ __launch_bounds__(256, (kWaves<E, DK>)) void delta_forward_kernel(DeltaP p) {
  typedef LdsIO<E> IO;
  constexpr bool TRANSFER = MODE == kTransfer, KEEP = MODE == kKeep;
  typedef ForwardChunk<E, DK, TRANSFER> Chunk;
  constexpr int PITCH = Chunk::PITCH, VP = Chunk::VP, KB = DK / 16, KS = DK / 32;
  extern __shared__ __align__(16) char smem[];
  Chunk& ch = *(Chunk*)smem;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, seg = blockIdx.z;
  const bool unit = TRANSFER && blockIdx.y < DK / 64;  // columns of the identity
  const int base = ((int)blockIdx.y - (TRANSFER && !unit ? DK / 64 : 0)) * 64, col0 = base + w * 16, col = col0 + l16;
  const bool mine = unit || col0 < p.dvp, on = unit || col < p.dv;  // (a wave past the columns only helps staging)
  const int len = delta_len(p, b), chunks = (len + kChunk - 1) / kChunk;
  const int c0 = seg * p.seg_chunks, c1 = min(c0 + p.seg_chunks, chunks);
  // (no segment enters behind the last; its X is the backward's all the same)
  if (TRANSFER && (unit && p.u ? c0 >= chunks : c1 >= chunks)) return;
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* qb = (const E*)p.q.ptr + b * p.q.sb + (h / p.rep) * p.q.sh;
  const E* vb = (const E*)p.v.ptr + b * p.v.sb + h * p.v.sh + (unit ? 0 : base);
  E* ob = (E*)p.out.ptr + b * p.out.sb + h * p.out.sh + col0 + 4 * g;
  const bool out_on = col0 + 4 * g < p.dv;

  floatx4 S[KB];
#pragma unroll
  for (int d = 0; d < KB; ++d) {
    S[d] = zero4();
    if (TRANSFER) {
      if (unit)
#pragma unroll
        for (int i = 0; i < 4; ++i) S[d][i] = 16 * d + 4 * g + i == col ? 1.f : 0.f;
    } else if (p.nseg > 1) {
      if (mine && (c0 < chunks || seg == 0))
        S[d] = *(const floatx4*)(p.seg_state + ((int64_t)bh * p.nseg + seg) * p.dvp * DK +
                                 block_at<DK>(col0 / 16, d, lane));
    } else if (p.state && on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * d + 4 * g + i;
        if (row < p.dk) S[d][i] = p.state[((int64_t)bh * p.dk + row) * p.dv + col];
      }
    }
  }
  ChunkTile<E, DK, 256> kt, qt;
  ChunkTile<E, 64, 256> vt;
  TriTile<3> tt, tp;
  const int vcols = unit ? 0 : p.dv - base;
  float vv = 0.f;
  kt.init(p.k.st, p.dk, tid);
  qt.init(p.q.st, p.dk, tid);
  vt.init(p.v.st, vcols, tid);
  auto fetch = [&](int c) {
    const int t0 = c * kChunk;
    const float* prep = p.prep + ((int64_t)bh * p.nc + c) * kRecord;
    kt.fetch(kb, p.k.st, t0, len);
    vt.fetch(vb, p.v.st, t0, len);
    tt.fetch(prep, tid);
    vv = prep[2 * kTriElems + min(tid, kVec - 1)];
    if (!TRANSFER) {
      qt.fetch(qb, p.q.st, t0, len);
      tp.fetch(prep + kTriElems, tid);
    }
  };
  if (c0 < c1) fetch(c0);
  loads_landed();
  for (int c = c0; c < c1; ++c) {
    const int t0 = c * kChunk;
    __syncthreads();  // the last chunk has been read
    kt.store(ch.k, PITCH, p.dk, tid);
    vt.store(ch.v, VP, vcols, tid);
    tt.store(ch.t, tid);
    ch.vec[tid] = vv;
    if (!TRANSFER) {
      qt.store(ch.q, PITCH, p.dk, tid);
      tp.store(ch.p, tid);
    }
    fetch(min(c + 1, c1 - 1));
    __syncthreads();
    if (!mine) continue;
    const E *ks = ch.k, *qs = ch.q;
    const int64_t n = (int64_t)bh * p.nc + c;
    const E *tri_t = ch.t, *tri_p = ch.p;
    const float* vec = ch.vec;

    // K S0 and S0^T Q^T (lane l16 a token, four columns): independent products side by side
    floatx4 R[4], O[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) R[r] = O[r] = zero4();
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const Parts<E, 3> sf(S[2 * s], S[2 * s + 1]);
      if constexpr (KEEP) {
        E* s0 = (E*)p.s0 + (n * p.dvp + col) * DK + 32 * s + 4 * g;
        sf.store2(s0, s0 + 16, p.s0_low);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        R[r] = mma_parts(row_perm<E>(ks + (16 * r + l16) * PITCH, s, g), sf, R[r]);
        if constexpr (!TRANSFER) O[r] = mma_parts(sf, row_perm<E>(qs + (16 * r + l16) * PITCH, s, g), O[r]);
      }
    }
    // R = b (V - e^G K S0)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const floatx4 eg = *(const floatx4*)(vec + 16 * r + 4 * g);
      const floatx4 be = *(const floatx4*)(vec + 2 * kChunk + 16 * r + 4 * g);
      const floatx4 v = col4<E>(ch.v, VP, 16 * r, 16 * w, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) R[r][i] = be[i] * fmaf(-eg[i], R[r][i], v[i]);
    }
    // (from a column's first row that is not finite on, its rows are left out of the products,
    // and what they would have reached is NaN: outputs behind, what is kept, and the state)
    bool spoilt = false;
    int first = kChunk;
    if constexpr (!TRANSFER) {
      float off = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) off = taint(R[r][i], off);
      spoilt = __any(off != off);
      if (spoilt) {
#pragma unroll
        for (int r = 3; r >= 0; --r)
#pragma unroll
          for (int i = 3; i >= 0; --i)
            if (R[r][i] * 0.f != 0.f) first = 16 * r + 4 * g + i;
        first = min(first, __shfl_xor(first, 16, 64));
        first = min(first, __shfl_xor(first, 32, 64));
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * r + 4 * g + i >= first) R[r][i] = 0.f;
      }
    }
    // U = Ti R
    floatx4 U[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) U[r] = zero4();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const Parts<E, 3> rf(R[2 * s], R[2 * s + 1]);
#pragma unroll
      for (int r = 2 * s; r < 4; ++r) U[r] = mma_parts(get_tri<3>(tri_t, r, s, lane), rf, U[r]);
    }
    // S = e^{G_63} S0 + K^T (e^{G_63 - G} U), and beside it O^T = e^G S0^T Q^T + U^T P^T
    const float whole = vec[3 * kChunk];
#pragma unroll
    for (int d = 0; d < KB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[d][i] *= whole;
    if constexpr (!TRANSFER) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float eg = vec[16 * r + l16];
#pragma unroll
        for (int i = 0; i < 4; ++i) O[r][i] *= eg;
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      floatx4 f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const floatx4 tail = *(const floatx4*)(vec + kChunk + 16 * (2 * s + e) + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[e][i] = U[2 * s + e][i] * tail[i];
      }
      const Parts<E, 3> ff(f[0], f[1]), uf(U[2 * s], U[2 * s + 1]);
      if constexpr (KEEP) {
        E* u = (E*)p.u + (n * p.dvp + col) * kChunk + 32 * s + 4 * g;
        uf.store2(u, u + 16, p.u_low);
      }
#pragma unroll
      for (int d = 0; d < KB; ++d) S[d] = mma_parts(TokFrag<E>::get(ks, PITCH, 16 * d, s, lane), ff, S[d]);
      if constexpr (!TRANSFER) {
#pragma unroll
        for (int r = 2 * s; r < 4; ++r) O[r] = mma_parts(uf, get_tri<3>(tri_p, r, s, lane), O[r]);
      }
    }
    if (spoilt) {
      const float nan = __builtin_nanf("");
      if (first < kChunk)
#pragma unroll
        for (int d = 0; d < KB; ++d) S[d] = floatx4{nan, nan, nan, nan};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int from = __shfl(first, 4 * g + i, 64);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * r + l16 >= from) O[r][i] = nan;
      }
      if constexpr (KEEP) {
        E* u = (E*)p.u + (n * p.dvp + col) * kChunk + 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * r + 4 * g + i >= first) u[16 * r + i] = (E)nan;
      }
    }
    if constexpr (!TRANSFER) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = t0 + 16 * r + l16;
        const bool in = t < len;
        if (t < p.T && out_on)
          IO::st4(ob + (int64_t)t * p.out.st, in ? O[r][0] : 0.f, in ? O[r][1] : 0.f, in ? O[r][2] : 0.f,
                  in ? O[r][3] : 0.f);
      }
    }
  }
  if (!mine) return;
  if constexpr (TRANSFER) {
    float* x = p.seg_x + ((int64_t)bh * p.nseg + seg) * p.seg_stride;
    const int cb = col0 / 16;
    if (!unit) {
#pragma unroll
      for (int d = 0; d < KB; ++d) *(floatx4*)(x + DK * DK + block_at<DK>(cb, d, lane)) = S[d];
      return;
    }
    // as operands of the segments' products: a row's columns in accumulator order (over
    // LDS, a wave its own columns'), and a column's rows
    constexpr int TP = DK + 4;
    static_assert(sizeof(Chunk) >= 4 * 16 * TP * sizeof(float), "columns of four waves");
    float* t = (float*)smem + w * 16 * TP;
    __syncthreads();  // the last chunk has been read
#pragma unroll
    for (int d = 0; d < KB; ++d) *(floatx4*)(t + l16 * TP + 16 * d + 4 * g) = S[d];
    wave_lds_sync();
#pragma unroll
    for (int d = 0; d < KB; ++d) {
      floatx4 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = t[(4 * g + j) * TP + 16 * d + l16];
      *(floatx4*)(x + ((d * KS + (cb >> 1)) * 64 + lane) * 8 + 4 * (cb & 1)) = r;
    }
    if (p.u)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        *(floatx8*)(x + (DK + p.dvp) * DK + ((cb * KS + s) * 64 + lane) * 8) =
            __builtin_shufflevector(S[2 * s], S[2 * s + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    return;
  }
  // tokens behind the length (those of its own chunk are written above), by the segment of each
  const int last = min(p.T, (c0 + p.seg_chunks) * kChunk);
  for (int t = max(c0, chunks) * kChunk + l16; t < last; t += 16)
    if (out_on) IO::st4(ob + (int64_t)t * p.out.st, 0.f, 0.f, 0.f, 0.f);
  // the segment that holds the last token (the first, where there is none) has the final state
  const bool final = chunks ? c0 < chunks && c0 + p.seg_chunks >= chunks : seg == 0;
  if (p.state_out && on && final) {
#pragma unroll
    for (int d = 0; d < KB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * d + 4 * g + i;
        if (row < p.dk) p.state_out[((int64_t)bh * p.dk + row) * p.dv + col] = S[d][i];
      }
  }
}

// The states entering the segments: S_{s+1} = X_s S_s + N_s for 16 value columns,
// a wave for every 16 rows, on fp32 MFMA.  BACK: dS_s = X_s^T dS_{s+1} + N_s from
// the last segment that any token reaches.  A step needs the whole state of the one
// before (through LDS); its matrices are loaded two steps ahead, whole lines at a time
// (31 steps of 64 keys 18.8 us, a step ahead 20.7, with X by column 26.7; three ahead 18.1,
// but spilled with 128 keys: seven steps 24 us against 17).
template <int DK, bool BACK>
__global__ __launch_bounds__(4 * DK, 4) void delta_segments_kernel(DeltaP p) {
  constexpr int KS = DK / 32, PITCH = DK + 4, AHEAD = 2;
  __shared__ __align__(16) float state[2][16 * PITCH];  // [column][row]
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x, b = bh / p.H, col = (int)blockIdx.y * 16 + l16;
  const int chunks = (delta_len(p, b) + kChunk - 1) / kChunk, segs = (chunks + p.seg_chunks - 1) / p.seg_chunks;
  const float* first = BACK ? p.dstate_out : p.state;
  floatx4 S = zero4();  // rows 16w + 4g ..
  if (first && col < p.dv) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * w + 4 * g + i;
      if (row < p.dk) S[i] = first[((int64_t)bh * p.dk + row) * p.dv + col];
    }
  }
  // the forward's first segment too enters from here: its own reading of the state
  // could meet the last segment's writing of its successor in place
  const int at_block = block_at<DK>((int)blockIdx.y, w, lane);
  if (!BACK) *(floatx4*)(p.seg_state + (int64_t)bh * p.nseg * p.dvp * DK + at_block) = S;
  const int steps = segs - 1;
  if (steps < 1) return;
  floatx8 xf[AHEAD][KS];  // row 16w + l16 of X (BACK: of X^T), columns in accumulator order
  floatx4 nf[AHEAD];
  auto load = [&](int k, floatx8* x8, floatx4& n4) {
    k = min(k, steps - 1);
    const int64_t at = (int64_t)bh * p.nseg + (BACK ? segs - 1 - k : k);
    const float* x = p.seg_x + at * p.seg_stride;
    n4 = *(const floatx4*)((BACK ? p.seg_n + at * p.dvp * DK : x + DK * DK) + at_block);
    if (BACK) x += (DK + p.dvp) * DK;
#pragma unroll
    for (int e = 0; e < KS; ++e) x8[e] = *(const floatx8*)(x + ((w * KS + e) * 64 + lane) * 8);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(i, xf[i], nf[i]);
  for (int k0 = 0; k0 < steps; k0 += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int k = k0 + i;
      if (i && k >= steps) break;  // uniform
      float* st = state[k & 1];
      *(floatx4*)(st + l16 * PITCH + 16 * w + 4 * g) = S;
      __syncthreads();
      S = nf[i];
#pragma unroll
      for (int e = 0; e < KS; ++e) S = mma32(xf[i][e], row_perm<float>(st + l16 * PITCH, e, g), S);
      load(k + AHEAD, xf[i], nf[i]);
      const int to = BACK ? segs - 2 - k : k + 1;
      *(floatx4*)(p.seg_state + ((int64_t)bh * p.nseg + to) * p.dvp * DK + at_block) = S;
    }
  }
}

template __global__ void delta_segments_kernel<64, true>(DeltaP);
template __global__ void delta_segments_kernel<128, true>(DeltaP);

// Segments of a sequence's chunks, one chain each.  A chain's chunks follow one
// another, so where heads and value columns alone leave CUs without a workgroup, the
// sequence is cut: every segment but the last first forms what it makes of its entering
// state (the transfer: dk more columns, no outputs), then the segments run side by side.
// n segments of nc / n chunks take n steps between them and 2 nc / n chunks of a chain:
// best near n^2 = c nc.  Measured (forward, 64 keys, operands in two parts): 8 heads of 1024 tokens 53 us
// whole, 38 at four segments, 32 at eight, of 4096 65 at eight, 55 at 16, 61 at 32:
// c = 4.  Where that is more than a workgroup a CU, chains side by side slow each other
// and c = 2: 64 heads of 1024 tokens 61 whole, 51 at four, 53 at eight; 8 of 32768 170
// at 16, 123 at 32, 129 at 64.  Two workgroups a CU at most.  Whole stay: five chunks and fewer
// (four: 23.5 us, in two segments 25.9); with more than 64 chains, under 32 chunks (128
// heads of 512 tokens 42 us, 47 in two, of 1024 68 and 70, of 2048 125 and in four 118);
// more than 128 chains (160 heads of 2048 tokens 143, 152 in three).
int delta_segments(const ts_delta_desc* d) {
  const int64_t chains = (int64_t)d->B * d->H * ((d->dv + 63) / 64);
  const int64_t nc = (d->T + kChunk - 1) / kChunk;
  if (nc < 6 || chains > 128 || (chains > 64 && nc < 32)) return 1;
  auto root = [](int64_t x) {
    int64_t n = 1;
    while ((n + 1) * (n + 1) <= x) ++n;
    return n;
  };
  int64_t n = root(4 * nc);
  if (n * chains > 256) n = root(2 * nc);
  if (n > 512 / chains) n = 512 / chains;
  if (n > nc / 2) n = nc / 2;
  const int64_t each = (nc + n - 1) / n;
  return (int)((nc + each - 1) / each);
}

int delta_check(const ts_delta_desc* d, const ts_delta_io* io, DeltaP* p, const char* what) {
  if (!d || d->B < 1 || d->Hk < 1 || d->H < 1 || d->H % d->Hk || d->T < 0 || d->dk < 1 || d->dv < 1)
    return fail(TS_ERR_VALUE, "%s: bad shape", what);
  if (d->dtype != TS_BF16 && d->dtype != TS_F32) return fail(TS_ERR_NOT_IMPLEMENTED, "%s: bf16 or fp32 only", what);
  const int vec = d->dtype == TS_BF16 ? 8 : 4;
  if (d->dk > 128 || d->dv > 512)
    return fail(TS_ERR_NOT_IMPLEMENTED, "%s: at most 128 keys and 512 values, got %d and %d", what, d->dk, d->dv);
  if (d->dk % vec || d->dv % vec) return fail(TS_ERR_VALUE, "%s: widths must be multiples of 16 bytes", what);
  // (a launch counts its threads in 32 bits: 256 to a head)
  if ((int64_t)d->B * d->H >= 1 << 24 || d->T > 0x7fffffff - 64)
    return fail(TS_ERR_NOT_IMPLEMENTED, "%s: too many heads or tokens", what);
  if (!p) return TS_OK;
  memset(p, 0, sizeof(*p));
  p->B = d->B; p->Hk = d->Hk; p->H = d->H; p->rep = d->H / d->Hk; p->T = d->T; p->dk = d->dk; p->dv = d->dv;
  p->nc = (d->T + kChunk - 1) / kChunk;
  p->dvp = (d->dv + 15) / 16 * 16;
  p->nseg = delta_segments(d);
  p->seg_chunks = (p->nc + p->nseg - 1) / p->nseg;
  p->beta_bf16 = d->beta_dtype == TS_BF16;
  p->decay_bf16 = d->decay_dtype == TS_BF16;
  if (!io) return TS_OK;
  auto rows = [&](const ts_strided& s) {
    return s.ptr && ((uintptr_t)s.ptr & 15u) == 0 && s.sb % vec == 0 && s.sh % vec == 0 && s.st % vec == 0;
  };
  if (!rows(io->q) || !rows(io->k) || !rows(io->v) || !rows(io->out))
    return fail(TS_ERR_VALUE, "%s: q, k, v and out need 16-byte aligned rows", what);
  if (!io->beta.ptr) return fail(TS_ERR_VALUE, "%s: missing beta", what);
  // (a chunk's rows are addressed in 32 bits from its first)
  const int64_t reach = ((int64_t)1 << 31) / (ts::kChunk * (16 / vec));
  for (int64_t st : {io->q.st, io->k.st, io->v.st})
    if (st < 0 || st >= reach) return fail(TS_ERR_NOT_IMPLEMENTED, "%s: 64 rows must lie within 2 GiB", what);
  p->q = io->q; p->k = io->k; p->v = io->v; p->out = io->out; p->beta = io->beta; p->decay = io->decay;
  p->lengths = io->lengths; p->state = io->state; p->state_out = io->state_out;
  return TS_OK;
}

}  // namespace ts

namespace {

using ts::DeltaP;
using ts::fail;

int padded_keys(int dk) { return dk <= 64 ? 64 : 128; }

struct Sizes {
  size_t prep, seg_x, seg_state, u, s0;  // bytes of each part; u and s0 only where kept
  size_t low;                            // bytes of ts_delta_io.low
  size_t all(const ts_delta_desc* d) const { return prep + seg_x + seg_state + (d->keep ? u + s0 : 0); }
};
Sizes sizes(const ts_delta_desc* d) {
  const size_t es = d->dtype == TS_BF16 ? 2 : 4;
  const size_t n = (size_t)d->B * d->H * ((d->T + 63) / 64), dvp = (d->dv + 15) / 16 * 16;
  Sizes s;
  s.prep = n * ts::kRecord * sizeof(float);
  const size_t seg = (size_t)d->B * d->H * ts::delta_segments(d), dkp = padded_keys(d->dk);
  s.seg_x = s.seg_state = 0;
  if (ts::delta_segments(d) > 1) {
    s.seg_x = seg * ts::seg_floats((int)dkp, (int)dvp, d->keep) * sizeof(float);
    s.seg_state = seg * dvp * dkp * sizeof(float);
  }
  s.u = n * dvp * 64 * es;
  s.s0 = n * dvp * padded_keys(d->dk) * es;
  s.low = d->keep && d->dtype == TS_BF16 ? s.u + s.s0 : 0;
  return s;
}

template <typename E, int DK, int MODE>
int launch(const DeltaP& p, unsigned columns, hipStream_t stream) {
  const int lds = (int)sizeof(ts::ForwardChunk<E, DK, MODE == ts::kTransfer>);
  if (ts::ensure_lds_limit((const void*)ts::delta_forward_kernel<E, DK, MODE>, lds) != hipSuccess)
    return fail(TS_ERR_RUNTIME, "delta: LDS of %d bytes", lds);
  hipLaunchKernelGGL((ts::delta_forward_kernel<E, DK, MODE>), dim3((unsigned)(p.B * p.H), columns, (unsigned)p.nseg),
                     dim3(256), lds, stream, p);
  return TS_OK;
}

template <typename E, int DK>
int forward(const DeltaP& p, hipStream_t stream) {
  const int64_t n = (int64_t)p.B * p.H * p.nc;
  hipLaunchKernelGGL((ts::delta_prepare_kernel<E, DK>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, stream, p);
  const unsigned columns = (unsigned)((p.dvp + 63) / 64);
  if (p.nseg > 1) {
    const int rc = launch<E, DK, ts::kTransfer>(p, columns + DK / 64, stream);
    if (rc) return rc;
    hipLaunchKernelGGL((ts::delta_segments_kernel<DK, false>), dim3((unsigned)(p.B * p.H), (unsigned)(p.dvp / 16)),
                       dim3(4 * DK), 0, stream, p);
  }
  return p.u ? launch<E, DK, ts::kKeep>(p, columns, stream) : launch<E, DK, ts::kForward>(p, columns, stream);
}

}  // namespace

extern "C" {

int ts_delta_workspace_bytes(const ts_delta_desc* d, size_t* bytes) {
  const int rc = ts::delta_check(d, nullptr, nullptr, "delta");
  if (rc) return rc;
  const Sizes s = sizes(d);
  if (bytes) *bytes = s.all(d);
  return TS_OK;
}

int ts_delta_low_bytes(const ts_delta_desc* d, size_t* bytes) {
  const int rc = ts::delta_check(d, nullptr, nullptr, "delta");
  if (rc) return rc;
  if (bytes) *bytes = sizes(d).low;
  return TS_OK;
}

int ts_delta_fwd(const ts_delta_desc* d, const ts_delta_io* io, void* workspace, size_t workspace_bytes,
                 hipStream_t stream) {
  DeltaP p;
  if (!io) return fail(TS_ERR_VALUE, "delta: missing tensors");
  const int rc = ts::delta_check(d, io, &p, "delta");
  if (rc) return rc;
  if (d->T == 0) return TS_OK;
  const Sizes s = sizes(d);
  if (!workspace || ((uintptr_t)workspace & 15u) || workspace_bytes < s.all(d))
    return fail(TS_ERR_VALUE, "delta: the workspace is missing, misaligned or too small");
  if (((int64_t)p.B * p.H * p.nc + 3) / 4 > 0x7fffffff) return fail(TS_ERR_NOT_IMPLEMENTED, "delta: grid too large");
  p.prep = (float*)workspace;
  p.seg_x = (float*)((char*)workspace + s.prep);
  p.seg_stride = ts::seg_floats(padded_keys(p.dk), p.dvp, d->keep);
  p.seg_state = (float*)((char*)workspace + s.prep + s.seg_x);
  if (d->keep) {
    p.u = (char*)workspace + s.prep + s.seg_x + s.seg_state;
    p.s0 = (char*)p.u + s.u;
    if (s.low) {
      if (!io->low || ((uintptr_t)io->low & 15u))
        return fail(TS_ERR_VALUE, "delta: the low halves' buffer is missing or misaligned");
      p.u_low = ((char*)io->low - (char*)p.u) / 2;
      p.s0_low = ((char*)io->low + s.u - (char*)p.s0) / 2;
    }
  }
  const bool narrow = d->dk <= 64;
  int rc2;
  if (d->dtype == TS_BF16)
    rc2 = narrow ? forward<ts::bf16, 64>(p, stream) : forward<ts::bf16, 128>(p, stream);
  else
    rc2 = narrow ? forward<float, 64>(p, stream) : forward<float, 128>(p, stream);
  if (rc2) return rc2;
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "delta: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}

}  // extern "C"
