// Gated delta rule, backward (gfx950); notation of ts_delta.h, X' the gradient
// of X, dS the gradient of the state behind a chunk.
//
//   dU = P^T dO + e^{G_63 - G} K dS,   dR = Ti^T dU,   dV = b dR
//   dS0 = e^{G_63} dS + Q^T (e^G dO) - K^T (b e^G dR)
//   A = e^{G_t - G_i} (dO U^T)_ti (i <= t),   M = -b e^{G_t - G_i} (dR U^T)_ti (i < t)
//   dQ = A K + e^G dO S0^T
//   dK = A^T Q + (M + M^T) K + e^{G_63 - G} U dS^T - b e^G dR S0^T
//   db_t = dR_t.U_t / b_t,   or dR_t.(v_t - e^{G_t} S0^T k_t - sum_i e^{G_t - G_i} k_t.k_i U_i) where b_t = 0
//   dlog a_t = sum_{i < t <= s} X_si + sum_{s >= t} h_s + sum_{i < t} f_i + e^{G_63} <S0, dS>,
//     X = A (Q K^T) + M (K K^T) elementwise,  h_s = e^{G_s} q_s.(S0 dO_s) - b e^{G_s} k_s.(S0 dR_s),
//     f_i = e^{G_63 - G_i} k_i.(dS U_i)
// (what token t's retention acts on, and nothing that would have to cancel: every term of a
// reset holds its zero, and a first token's without an entering state are none.)
//
// delta_chain walks the chunks backwards, a wave per 16 value columns as in the
// forward; it leaves dR and dS per chunk and writes dV.  delta_grads takes the
// chunks on their own: one workgroup each, a wave per 16 tokens.
//
// Roundings (bf16 inputs): every operand that is not an input is a pair of bf16 parts, 16 bits,
// also as kept (U, S0, dR, dS), since sums over alike keys cancel: with these rounded once
// the gradients of 256 nearly alike keys were off by 0.8 % (dq), 0.5 (dv), 0.8 (db) and 1.0 (the
// retentions'), of one key throughout up to 7 % (float64 emulation), with the pairs 1e-5.  A
// bf16 gradient's own rounding is 0.0017 of it; fp32 ones (of states and fp32 gates) hold
// those 16 bits, 3e-6 to 5e-5.  Sums are fp32, those of the gates' gradients over a chunk fp64.
//
// 64 heads of 4096 tokens of 64 x 64, bf16 (bytes by counters): transfers 48 us (187 MB), chain
// 95 (390 MB, 4.1 TB/s), gradients 116 to 123 (495 MB, 4.0 to 4.3 TB/s; its loads and its products
// take turns in a workgroup, three of which share a CU).  Without the low halves 33, 62 and 80 us.

#include "ts_delta.h"

#include <string.h>

#include <type_traits>

namespace ts {

// What the waves of a workgroup read of one chunk.
template <typename E, int DK>
struct ChainChunk {
  static constexpr int PAD = 16 / (int)sizeof(E), PITCH = DK + PAD, VP = 64 + PAD, SET = kParts<E, 2> * kTriElems;
  E k[kChunk * PITCH], q[kChunk * PITCH], o[kChunk * VP], t[SET], p[SET];
  float vec[256];
};
// TRANSFER: what a segment of chunks adds to the gradient behind it, from its
// tokens alone (X^T of the forward's transfer makes the rest): nothing is stored
// but that.
template <typename E, int DK, bool TRANSFER>
__global__ __launch_bounds__(256, (kWaves<E, DK>)) void delta_chain_kernel(DeltaP p) {
  typedef LdsIO<E> IO;
  typedef typename Frag<E>::f8 f8;
  typedef ChainChunk<E, DK> Chunk;
  constexpr int PITCH = Chunk::PITCH, VP = Chunk::VP, KB = DK / 16, KS = DK / 32;
  extern __shared__ __align__(16) char smem[];
  Chunk& lds = *(Chunk*)smem;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, seg = blockIdx.z;
  const int base = (int)blockIdx.y * 64, col0 = base + w * 16, col = col0 + l16;
  const bool mine = col0 < p.dvp, on = col < p.dv;
  const int len = delta_len(p, b), chunks = (len + kChunk - 1) / kChunk;
  const int c0 = seg * p.seg_chunks, c1 = min(c0 + p.seg_chunks, chunks);
  if (TRANSFER && (seg == 0 || c0 >= chunks)) return;  // (nothing is behind it to hand it on to)
  // the segment of the last token (the first, where there is none) starts from the final state's gradient
  const bool final = chunks ? c0 < chunks && c0 + p.seg_chunks >= chunks : seg == 0;
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* qb = (const E*)p.q.ptr + b * p.q.sb + (h / p.rep) * p.q.sh;
  const E* db = (const E*)p.dout.ptr + b * p.dout.sb + h * p.dout.sh + base;
  E* vb = (E*)p.dval.ptr + b * p.dval.sb + h * p.dval.sh + col;

  floatx4 S[KB];  // dS
#pragma unroll
  for (int d = 0; d < KB; ++d) {
    S[d] = zero4();
    if (TRANSFER) continue;
    if (!final) {
      if (mine && c0 < chunks)
        S[d] = *(const floatx4*)(p.seg_state + ((int64_t)bh * p.nseg + seg) * p.dvp * DK +
                                 block_at<DK>(col0 / 16, d, lane));
    } else if (p.dstate_out && on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * d + 4 * g + i;
        if (row < p.dk) S[d][i] = p.dstate_out[((int64_t)bh * p.dk + row) * p.dv + col];
      }
    }
  }
  ChunkTile<E, DK, 256> kt, qt;
  ChunkTile<E, 64, 256> ot;
  kt.init(p.k.st, p.dk, tid);
  qt.init(p.q.st, p.dk, tid);
  ot.init(p.dout.st, p.dv - base, tid);
  TriTile<2> tt, tp;
  float vv = 0.f;
  auto fetch = [&](int c) {
    const int t0 = c * kChunk;
    kt.fetch(kb, p.k.st, t0, len);
    qt.fetch(qb, p.q.st, t0, len);
    ot.fetch(db, p.dout.st, t0, len);
    const float* prep = p.prep + ((int64_t)bh * p.nc + c) * kRecord;
    tt.fetch(prep, tid);
    tp.fetch(prep + kTriElems, tid);
    vv = prep[2 * kTriElems + min(tid, kVec - 1)];
  };
  if (c0 < c1) fetch(c1 - 1);
  loads_landed();
  for (int c = c1 - 1; c >= c0; --c) {
    const int t0 = c * kChunk;
    const int64_t n = (int64_t)bh * p.nc + c;
    __syncthreads();  // the last chunk has been read
    kt.store(lds.k, PITCH, p.dk, tid);
    qt.store(lds.q, PITCH, p.dk, tid);
    ot.store(lds.o, VP, p.dv - base, tid);
    tt.store(lds.t, tid);
    tp.store(lds.p, tid);
    lds.vec[tid] = vv;
    fetch(max(c - 1, c0));
    __syncthreads();
    if (!mine) continue;
    const float* vec = lds.vec;
    f8 of[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) of[s] = TokFrag<E>::get(lds.o, VP, 16 * w, s, lane);

    // dU = P^T dO + e^{G_63 - G} K dS, and beside it Q^T (e^G dO): independent products
    floatx4 X[4], Y[4], Z[KB];
#pragma unroll
    for (int r = 0; r < 4; ++r) X[r] = Y[r] = zero4();
#pragma unroll
    for (int d = 0; d < KB; ++d) Z[d] = zero4();
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const Parts<E, 2> sf(S[2 * s], S[2 * s + 1]);
      if constexpr (!TRANSFER) {
        E* ds = (E*)p.ds + (n * p.dvp + col) * DK + 32 * s + 4 * g;
        sf.store2(ds, ds + 16, p.ds_low);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) X[r] = mma_parts(row_perm<E>(lds.k + (16 * r + l16) * PITCH, s, g), sf, X[r]);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      floatx4 f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const floatx4 eg = *(const floatx4*)(vec + 16 * (2 * s + e) + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[e][i] = eg[i] * tof(of[s][4 * e + i]);
      }
      const Parts<E, 2> qf(f[0], f[1]);
#pragma unroll
      for (int r = 0; r < 2 * s + 2; ++r) Y[r] = mma_parts(get_tri_t<2>(lds.p, r, s, lane), of[s], Y[r]);
#pragma unroll
      for (int d = 0; d < KB; ++d) Z[d] = mma_parts(TokFrag<E>::get(lds.q, PITCH, 16 * d, s, lane), qf, Z[d]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const floatx4 tail = *(const floatx4*)(vec + kChunk + 16 * r + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) X[r][i] = fmaf(tail[i], X[r][i], Y[r][i]);
    }
    // dR = Ti^T dU
    floatx4 R[4];
    {
      const Parts<E, 2> u0(X[0], X[1]), u1(X[2], X[3]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        R[r] = mma_parts(get_tri_t<2>(lds.t, r, 1, lane), u1, zero4());
        if (r < 2) R[r] = mma_parts(get_tri_t<2>(lds.t, r, 0, lane), u0, R[r]);
      }
    }
    if constexpr (!TRANSFER) {
      E* dro = (E*)p.dr + (n * p.dvp + col) * kChunk + 4 * g;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        Parts<E, 2>(R[2 * s], R[2 * s + 1]).store2(dro + 32 * s, dro + 32 * s + 16, p.dr_low);
    }
    const float whole = vec[3 * kChunk];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const floatx4 eg = *(const floatx4*)(vec + 16 * r + 4 * g);
      const floatx4 be = *(const floatx4*)(vec + 2 * kChunk + 16 * r + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + 16 * r + 4 * g + i;
        const float dv = be[i] * R[r][i];
        if (!TRANSFER && t < p.T && on) vb[(int64_t)t * p.dval.st] = cvt<E>(t < len ? dv : 0.f);
        R[r][i] = -eg[i] * dv;
      }
    }
    // dS0
#pragma unroll
    for (int d = 0; d < KB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[d][i] = fmaf(whole, S[d][i], Z[d][i]);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const Parts<E, 2> rf(R[2 * s], R[2 * s + 1]);
#pragma unroll
      for (int d = 0; d < KB; ++d) S[d] = mma_parts(TokFrag<E>::get(lds.k, PITCH, 16 * d, s, lane), rf, S[d]);
    }
  }
  if (!mine) return;
  if constexpr (TRANSFER) {
    float* nn = p.seg_n + ((int64_t)bh * p.nseg + seg) * p.dvp * DK;
#pragma unroll
    for (int d = 0; d < KB; ++d) *(floatx4*)(nn + block_at<DK>(col0 / 16, d, lane)) = S[d];
    return;
  }
  const int last = min(p.T, (c0 + p.seg_chunks) * kChunk);
  if (on)
    for (int t = max(c0, chunks) * kChunk + g; t < last; t += 4) vb[(int64_t)t * p.dval.st] = (E)0.0f;
  if (p.dstate && on && seg == 0) {
#pragma unroll
    for (int d = 0; d < KB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * d + 4 * g + i;
        if (row < p.dk) p.dstate[((int64_t)bh * p.dk + row) * p.dv + col] = S[d][i];
      }
  }
}

// Value columns of a pass of delta_grads.
constexpr int kGradCols = 32;

template <typename E, int DK>
struct GradsLds {
  static constexpr int PAD = 16 / (int)sizeof(E), PITCH = DK + PAD, VB = kGradCols, TP = kChunk + PAD;
  static constexpr int N = kParts<E, 2>, US = VB * TP, SS = VB * PITCH;  // elements of one of a pair's halves
  struct Pass {
    E u[N * US], dr[N * US], s0[N * SS], ds[N * SS];
  };
  struct Pairs {
    E q[kChunk * PITCH], a[N * kTriElems], m[N * kTriElems];
  };
  E k[kChunk * PITCH];
  union {  // the passes over the value columns, then the pairs of tokens
    Pass pass;
    Pairs pairs;
  };
  double G[kChunk];
  float cols[4][kChunk], base[kChunk], f[kChunk], red[4];
};

// The sum over the 16 lanes of a row, in each of them.
__device__ __forceinline__ float row_sum(float x) {
  auto add = [&](auto ctrl) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xb1>());   // lanes 1, 0, 3, 2
  add(std::integral_constant<int, 0x4e>());   // lanes 2, 3, 0, 1
  add(std::integral_constant<int, 0x141>());  // the half row mirrored
  add(std::integral_constant<int, 0x140>());  // the row mirrored
  return x;
}

// Eight columns of a global row in accumulator order (c.., c + 16..), zero at or
// past `width` and where the row is none.
template <typename E>
__device__ __forceinline__ typename Frag<E>::f8 row_global(const E* row, int c, int width, bool on) {
  typename Frag<E>::f4 part[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool in = c + 16 * i < width;
    part[i] = LdsIO<E>::ld4(row + (in ? c + 16 * i : 0));
    if (!(in && on))
#pragma unroll
      for (int j = 0; j < 4; ++j) part[i][j] = (E)0.0f;
  }
  return LdsIO<E>::cat(part[0], part[1]);
}

// [ROWS x W] contiguous rows (of pairs: `low` elements from one half to the other) on their
// way to LDS; rows at or past `rows` are zero.
template <typename E, int ROWS, int W>
struct Block {
  static constexpr int VEC = 16 / (int)sizeof(E), PER = W / VEC, SLOTS = ROWS * PER / 256, N = kParts<E, 2>;
  uint4 r[N][SLOTS];
  __device__ __forceinline__ void fetch(const E* src, int64_t low, int rows, int tid) {
#pragma unroll
    for (int h = 0; h < N; ++h)
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        const int idx = tid + i * 256;
        r[h][i] = *(const uint4*)(src + h * low + min(idx / PER, rows - 1) * W + (idx % PER) * VEC);
      }
  }
  __device__ __forceinline__ void store(E* dst, int rows, int pitch, int tid) {
    if (rows < ROWS) {  // uniform
#pragma unroll
      for (int h = 0; h < N; ++h)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
          if ((tid + i * 256) / PER >= rows) r[h][i] = make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int h = 0; h < N; ++h)
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        const int idx = tid + i * 256;
        *(uint4*)(dst + (h * ROWS + idx / PER) * pitch + (idx % PER) * VEC) = r[h][i];
      }
  }
  // Sum of the products with another block's entries of the same places.
  __device__ __forceinline__ float dot(const Block& o) const {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      Vec16<E> a[N], b[N];
#pragma unroll
      for (int h = 0; h < N; ++h) {
        a[h].raw = r[h][i];
        b[h].raw = o.r[h][i];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum = fmaf(whole(a, j), whole(b, j), sum);
    }
    return sum;
  }
  static __device__ __forceinline__ float whole(const Vec16<E>* v, int j) {
    return N == 2 ? tof(v[0].e[j]) + tof(v[N - 1].e[j]) : tof(v[0].e[j]);
  }
};

// TokFrag of a tile of pairs, `half` elements from one half to the other.
template <typename E>
__device__ __forceinline__ Parts<E, 2> pair_frag(const E* rows, int half, int pitch, int c0, int kp, int lane) {
  Parts<E, 2> f;
#pragma unroll
  for (int i = 0; i < kParts<E, 2>; ++i) f.p[i] = TokFrag<E>::get(rows + i * half, pitch, c0, kp, lane);
  return f;
}

// (three waves a SIMD where registers and LDS allow it: without the low halves 102 us with two,
// 87 with three; the keys have a place of their own, in LDS from the first pass on and out of
// registers: 80)
template <typename E, int DK>
__global__ __launch_bounds__(256, (DK == 64 && sizeof(E) == 2 ? 3 : kWaves<E, DK>)) void delta_grads_kernel(DeltaP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  typedef GradsLds<E, DK> Lds;
  constexpr int PITCH = Lds::PITCH, VB = Lds::VB, TP = Lds::TP, US = Lds::US, SS = Lds::SS;
  constexpr int KB = DK / 16, KS = DK / 32;
  extern __shared__ __align__(16) char smem[];
  Lds& lds = *(Lds*)smem;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n = blockIdx.x;
  const int c = (int)(n % p.nc), bh = (int)(n / p.nc), b = bh / p.H, h = bh % p.H;
  const int t0 = c * kChunk, len = delta_len(p, b);
  const int64_t gate0 = (int64_t)bh * p.T + t0;
  const int t = 16 * w + l16;  // this lane's token of the chunk
  auto put_gate = [&](void* dst, int bf, int64_t i, float v) {
    if (bf)
      ((bf16*)dst)[i] = (bf16)v;
    else
      ((float*)dst)[i] = v;
  };
  // gradient rows of a token: columns 16d + 4g ..
  auto put_row = [&](const ts_strided& s, int d, const floatx4& v) {
    if (t0 + t >= p.T || 16 * d + 4 * g >= p.dk) return;
    const int64_t at = b * s.sb + h * s.sh + (int64_t)(t0 + t) * s.st + 16 * d + 4 * g;
    if (p.grad_f32)
      *(floatx4*)((float*)s.ptr + at) = v;
    else
      IO::st4((E*)s.ptr + at, v[0], v[1], v[2], v[3]);
  };
  if (t0 >= len) {  // a chunk behind the sequence
#pragma unroll
    for (int d = 0; d < KB; ++d) {
      put_row(p.dq, d, zero4());
      put_row(p.dkey, d, zero4());
    }
    if (tid < kChunk && t0 + tid < p.T) {
      put_gate(p.dbeta, p.beta_bf16, gate0 + tid, 0.f);
      if (p.ddecay) put_gate(p.ddecay, p.ddecay_bf16, gate0 + tid, 0.f);
    }
    return;
  }
  const E* kb = (const E*)p.k.ptr + b * p.k.sb + (h / p.rep) * p.k.sh;
  const E* qb = (const E*)p.q.ptr + b * p.q.sb + (h / p.rep) * p.q.sh;
  // every row of the first pass on its way at once
  ChunkTile<E, DK, 256> kt, qt;
  Block<E, VB, kChunk> ut, rt;
  Block<E, VB, DK> st, dt;
  f8 of[VB / 32];  // this wave's rows of dO
  const E* orow = (const E*)p.dout.ptr + b * p.dout.sb + h * p.dout.sh + (int64_t)min(t0 + t, len - 1) * p.dout.st;
  const E* vrow = (const E*)p.v.ptr + b * p.v.sb + h * p.v.sh + (int64_t)min(t0 + t, len - 1) * p.v.st;
  auto fetch = [&](int v0) {
    const int rows = p.dvp - v0;
#pragma unroll
    for (int s = 0; s < VB / 32; ++s) of[s] = row_global<E>(orow, v0 + 32 * s + 4 * g, p.dv, t0 + t < len);
    ut.fetch((const E*)p.u + (n * p.dvp + v0) * kChunk, p.u_low, rows, tid);
    rt.fetch((const E*)p.dr + (n * p.dvp + v0) * kChunk, p.dr_low, rows, tid);
    st.fetch((const E*)p.s0 + (n * p.dvp + v0) * DK, p.s0_low, rows, tid);
    dt.fetch((const E*)p.ds + (n * p.dvp + v0) * DK, p.ds_low, rows, tid);
  };
  kt.init(p.k.st, p.dk, tid);
  qt.init(p.q.st, p.dk, tid);
  kt.fetch(kb, p.k.st, t0, len);
  qt.fetch(qb, p.q.st, t0, len);
  fetch(0);
  const float* vec = p.prep + n * kRecord + 2 * kTriElems;
  const float eg = vec[t], tail = vec[kChunk + t], be = vec[2 * kChunk + t], whole = vec[3 * kChunk];
  if (w == 0) {
    double sum = 0.0;
    if (p.decay.ptr && t0 + lane < len) {
      const float la =
          gate_at(p.decay, p.decay_bf16, b * p.decay.sb + h * p.decay.sh + (int64_t)(t0 + lane) * p.decay.st);
      sum = la < -1000.f ? -1000.0 : (double)la;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double below = __shfl_up(sum, o, 64);
      if (lane >= o) sum += below;
    }
    lds.G[lane] = sum;
  }
  // where a token's b is zero, db takes its values' rows too
  const bool zero_b = t0 + t < len && fabsf(be) < 1e-30f;
  const bool any_zero = __any(zero_b);

  floatx4 dp[4], ru[4], z[KB], y[KB], fu[KB], rv = zero4();
#pragma unroll
  for (int r = 0; r < 4; ++r) dp[r] = ru[r] = zero4();
#pragma unroll
  for (int d = 0; d < KB; ++d) z[d] = y[d] = fu[d] = zero4();
  float inner = 0.f;  // this thread's part of <S0, dS>
  kt.clear(t0, len, tid);
  qt.clear(t0, len, tid);
  for (int v0 = 0; v0 < p.dvp; v0 += VB) {
    if (v0) {
      __syncthreads();  // the last pass has been read
      fetch(v0);
    }
    const int rows = p.dvp - v0;
    if (v0 == 0) kt.store(lds.k, PITCH, p.dk, tid);
    ut.store(lds.pass.u, rows, TP, tid);
    rt.store(lds.pass.dr, rows, TP, tid);
    st.store(lds.pass.s0, rows, PITCH, tid);
    dt.store(lds.pass.ds, rows, PITCH, tid);
    inner += st.dot(dt);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < VB / 32; ++s) {
      const Parts<E, 2> rf = pair_frag(lds.pass.dr, US, TP, 16 * w, s, lane);
      const Parts<E, 2> uw = pair_frag(lds.pass.u, US, TP, 16 * w, s, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r <= w) {
          const Parts<E, 2> uf = pair_frag(lds.pass.u, US, TP, 16 * r, s, lane);
          dp[r] = mma_parts(uf, of[s], dp[r]);
          ru[r] = mma_parts(uf, rf, ru[r]);
        }
#pragma unroll
      for (int d = 0; d < KB; ++d) {
        const Parts<E, 2> sf = pair_frag(lds.pass.s0, SS, PITCH, 16 * d, s, lane);
        z[d] = mma_parts(sf, of[s], z[d]);
        y[d] = mma_parts(sf, rf, y[d]);
        fu[d] = mma_parts(pair_frag(lds.pass.ds, SS, PITCH, 16 * d, s, lane), uw, fu[d]);
      }
      if (any_zero) {
        const f8 vf = row_global<E>(vrow, v0 + 32 * s + 4 * g, p.dv, t0 + t < len);
        rv = mma_parts(vf, rf, rv);
      }
    }
  }
  __syncthreads();  // the last pass has been read: keys, queries and pairs take its place
  qt.store(lds.pairs.q, PITCH, p.dk, tid);
  __syncthreads();
  // pairs (i, t): rows i = 16r + 4g + j, column t
  const double gt = lds.G[t];
  float rows_n = 0.f, before = 0.f;  // before: row t of X up to block r
  float cx[16];                      // X_t0 + .. + X_ti, i < t
#pragma unroll
  for (int i = 0; i < 16; ++i) cx[i] = 0.f;
  float diag = 0.f, diag_v = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r <= w) {
      floatx4 kk = zero4(), qk = zero4();
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const f8 ki = IO::ld8(lds.k + (16 * r + l16) * PITCH + 32 * s + 8 * g);
        kk = mma32(ki, IO::ld8(lds.k + t * PITCH + 32 * s + 8 * g), kk);
        qk = mma32(ki, IO::ld8(lds.pairs.q + t * PITCH + 32 * s + 8 * g), qk);
      }
      float own = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 16 * r + 4 * g + j;
        const float d = __builtin_amdgcn_exp2f((float)((gt - lds.G[i]) * kLog2e));
        if (i == t) {
          diag = ru[r][j];
          diag_v = rv[j];
        }
        const float a = i <= t ? dp[r][j] * d : 0.f, m = i < t ? ru[r][j] * d : 0.f;
        const float xn = m * kk[j];
        rows_n += xn;
        own += fmaf(-be, xn, i < t ? a * qk[j] : 0.f);
        cx[4 * r + j] = own;
        dp[r][j] = a;
        ru[r][j] = -be * m;
      }
      // the lanes of lower columns: pairs give the even row's value first, then the lower half's
      const LanePair near = xor16_pair(own), far = xor32_pair(near.a + near.b);
      const float below = before + ((g & 1 ? near.a : 0.f) + (g & 2 ? far.a : 0.f));
#pragma unroll
      for (int j = 0; j < 4; ++j) cx[4 * r + j] = 16 * r + 4 * g + j < t ? below + cx[4 * r + j] : 0.f;
      before += far.a + far.b;
    } else {
      dp[r] = ru[r] = zero4();
    }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    cx[i] = row_sum(cx[i]);
    if (l16 == 0) lds.cols[w][16 * (i >> 2) + 4 * g + (i & 3)] = cx[i];
  }
#pragma unroll
  for (int s = 0; s < 2; ++s)
    if (2 * s <= w) {
      put_tri(lds.pairs.a, w, s, lane, Parts<E, 2>(dp[2 * s], dp[2 * s + 1]));
      put_tri(lds.pairs.m, w, s, lane, Parts<E, 2>(ru[2 * s], ru[2 * s + 1]));
    }
  // state terms of the gates, and of the rows
  float zq = 0.f, yk = 0.f, fk = 0.f;
#pragma unroll
  for (int d = 0; d < KB; ++d) {
    float qv[4], kv[4];
    ld4f<E>(lds.pairs.q + t * PITCH + 16 * d + 4 * g, qv);
    ld4f<E>(lds.k + t * PITCH + 16 * d + 4 * g, kv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      zq = fmaf(z[d][i], qv[i], zq);
      yk = fmaf(y[d][i], kv[i], yk);
      fk = fmaf(fu[d][i], kv[i], fk);
      z[d][i] *= eg;
      fu[d][i] = fmaf(tail, fu[d][i], -be * eg * y[d][i]);
    }
  }
  zq = sum_g(zq) * eg;
  yk = sum_g(yk) * eg;
  fk = sum_g(fk) * tail;
  rows_n = sum_g(rows_n);
  if (g == 0) {
    lds.base[t] = zq - be * yk;
    lds.f[t] = fk;
  }
  if (g == (l16 >> 2) && t0 + t < p.T) {  // the lane that holds (t, t)
    const float v = t0 + t >= len ? 0.f : zero_b ? diag_v - yk - rows_n : diag / be;
    put_gate(p.dbeta, p.beta_bf16, gate0 + t, v);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) inner += __shfl_xor(inner, o, 64);
  if (lane == 0) lds.red[w] = inner;
  __syncthreads();
  // dQ^T = K^T A^T + .., dK^T = Q^T A + K^T (M + M^T)^T + ..
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (2 * s <= w) {
      const Parts<E, 2> af(dp[2 * s], dp[2 * s + 1]), mf(ru[2 * s], ru[2 * s + 1]);
#pragma unroll
      for (int d = 0; d < KB; ++d) {
        const f8 kf = TF::get(lds.k, PITCH, 16 * d, s, lane);
        z[d] = mma_parts(kf, af, z[d]);
        fu[d] = mma_parts(kf, mf, fu[d]);
      }
    }
    if (2 * s + 1 >= w) {
      const Parts<E, 2> at = get_tri_t<2>(lds.pairs.a, w, s, lane), mt = get_tri_t<2>(lds.pairs.m, w, s, lane);
#pragma unroll
      for (int d = 0; d < KB; ++d) {
        fu[d] = mma_parts(TF::get(lds.k, PITCH, 16 * d, s, lane), mt, fu[d]);
        fu[d] = mma_parts(TF::get(lds.pairs.q, PITCH, 16 * d, s, lane), at, fu[d]);
      }
    }
  }
  const bool in = t0 + t < len;
#pragma unroll
  for (int d = 0; d < KB; ++d) {
    put_row(p.dq, d, in ? z[d] : zero4());
    put_row(p.dkey, d, in ? fu[d] : zero4());
  }
  if (w == 0 && p.ddecay) {
    double behind = (double)lds.base[lane], ahead = lane ? (double)lds.f[lane - 1] : 0.0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double above = __shfl_down(behind, o, 64), below = __shfl_up(ahead, o, 64);
      if (lane + o < 64) behind += above;
      if (lane >= o) ahead += below;
    }
    double dg = behind + ahead + (double)whole * ((double)lds.red[0] + lds.red[1] + lds.red[2] + lds.red[3]);
    if (lane)
#pragma unroll
      for (int r = 0; r < 4; ++r) dg += (double)lds.cols[r][lane - 1];
    if (t0 + lane < p.T) put_gate(p.ddecay, p.ddecay_bf16, gate0 + lane, t0 + lane < len ? (float)dg : 0.f);
  }
}

// Rows of `rep` value heads added up, in head order: x [B,H,T,W] fp32
// contiguous -> out [B,H/rep,T,W], for the queries and (y = 1) the keys.  Bound by its
// bytes: 32 heads of 2048 tokens of 128, two to a key, 84 MB in 14.8 us (two launches took 17.6).
template <typename E>
__global__ __launch_bounds__(256) void delta_group_sum_kernel(const float* x, ts_strided dq, ts_strided dkey, int Hk,
                                                              int rep, int T, int W, int64_t total) {
  const ts_strided& out = blockIdx.y ? dkey : dq;
  if (blockIdx.y) x += total * rep * 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int cols = W / 4, c = (int)(i % cols) * 4;
    const int64_t row = i / cols;
    const int t = (int)(row % T);
    const int64_t bk = row / T;
    const int b = (int)(bk / Hk), hk = (int)(bk % Hk);
    floatx4 sum = zero4();
    for (int r = 0; r < rep; ++r) {
      const floatx4 v = *(const floatx4*)(x + ((bk * rep + r) * T + t) * W + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
    LdsIO<E>::st4((E*)out.ptr + b * out.sb + hk * out.sh + (int64_t)t * out.st + c, sum[0], sum[1], sum[2], sum[3]);
  }
}

// out[h] = sum over batch and time of x [B,H,T] (a static retention's gradient).
template <typename O>
__global__ __launch_bounds__(256) void delta_head_sum_kernel(const float* x, O* out, int B, int H, int T) {
  __shared__ double part[256];
  const int h = blockIdx.x, tid = threadIdx.x;
  double sum = 0.0;
  for (int b = 0; b < B; ++b) {
    const float* row = x + ((int64_t)b * H + h) * T;
    for (int t = tid; t < T; t += 256) sum += (double)row[t];
  }
  part[tid] = sum;
  __syncthreads();
  for (int o = 128; o >= 1; o >>= 1) {
    if (tid < o) part[tid] += part[tid + o];
    __syncthreads();
  }
  if (tid == 0) out[h] = (O)(float)part[0];
}

}  // namespace ts

namespace {

using ts::DeltaP;
using ts::fail;

template <typename E, int DK>
int backward(const DeltaP& p, hipStream_t stream) {
  const int chain = (int)sizeof(ts::ChainChunk<E, DK>), grads = (int)sizeof(ts::GradsLds<E, DK>);
  if (ts::ensure_lds_limit((const void*)ts::delta_chain_kernel<E, DK, false>, chain) != hipSuccess ||
      ts::ensure_lds_limit((const void*)ts::delta_chain_kernel<E, DK, true>, chain) != hipSuccess ||
      ts::ensure_lds_limit((const void*)ts::delta_grads_kernel<E, DK>, grads) != hipSuccess)
    return fail(TS_ERR_RUNTIME, "delta bwd: LDS of %d bytes", grads);
  const dim3 grid((unsigned)(p.B * p.H), (unsigned)((p.dvp + 63) / 64), (unsigned)p.nseg);
  if (p.nseg > 1) {
    hipLaunchKernelGGL((ts::delta_chain_kernel<E, DK, true>), grid, dim3(256), chain, stream, p);
    hipLaunchKernelGGL((ts::delta_segments_kernel<DK, true>), dim3((unsigned)(p.B * p.H), (unsigned)(p.dvp / 16)),
                       dim3(4 * DK), 0, stream, p);
  }
  hipLaunchKernelGGL((ts::delta_chain_kernel<E, DK, false>), grid, dim3(256), chain, stream, p);
  hipLaunchKernelGGL((ts::delta_grads_kernel<E, DK>), dim3((unsigned)((int64_t)p.B * p.H * p.nc)), dim3(256), grads,
                     stream, p);
  return TS_OK;
}

// The rows of value heads that share keys (fp32), added up.
template <typename E>
void group_sum(const DeltaP& p, const float* x, const ts_strided& dq, const ts_strided& dkey, hipStream_t stream) {
  const int64_t total = (int64_t)p.B * p.Hk * p.T * (p.dk / 4), blocks = (total + 255) / 256;
  hipLaunchKernelGGL((ts::delta_group_sum_kernel<E>), dim3((unsigned)(blocks < 4096 ? blocks : 4096), 2),
                     dim3(256), 0, stream, x, dq, dkey, p.Hk, p.rep, p.T, p.dk, total);
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace

extern "C" {

int ts_delta_bwd_workspace_bytes(const ts_delta_desc* d, size_t* bytes) {
  const int rc = ts::delta_check(d, nullptr, nullptr, "delta bwd");
  if (rc) return rc;
  const size_t n = (size_t)d->B * d->H * ((d->T + 63) / 64), dvp = (d->dv + 15) / 16 * 16;
  const size_t dkp = d->dk <= 64 ? 64 : 128, nseg = ts::delta_segments(d);
  size_t total = n * dvp * (64 + dkp) * sizeof(float);  // (dR and dS, fp32 or two bf16 each)
  if (nseg > 1) total += 2 * (size_t)d->B * d->H * nseg * dvp * dkp * sizeof(float);
  if (d->H != d->Hk) total += align16(2 * (size_t)d->B * d->H * d->T * d->dk * sizeof(float));
  if (bytes) *bytes = total + align16((size_t)d->B * d->H * d->T * sizeof(float));
  return TS_OK;
}

int ts_delta_bwd(const ts_delta_desc* d, const ts_delta_io* io, const ts_delta_grads* gr, const void* saved,
                 size_t saved_bytes, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  DeltaP p;
  if (!io || !gr) return fail(TS_ERR_VALUE, "delta bwd: missing tensors");
  int rc = ts::delta_check(d, io, &p, "delta bwd");
  if (rc) return rc;
  if (d->T == 0) return TS_OK;
  size_t need = 0, kept = 0;
  rc = ts_delta_bwd_workspace_bytes(d, &need);
  if (rc) return rc;
  ts_delta_desc whole = *d;
  whole.keep = 1;
  rc = ts_delta_workspace_bytes(&whole, &kept);
  if (rc) return rc;
  if (!saved || ((uintptr_t)saved & 15u) || saved_bytes < kept || !workspace || ((uintptr_t)workspace & 15u) ||
      workspace_bytes < need)
    return fail(TS_ERR_VALUE, "delta bwd: the saved buffer or the workspace is missing, misaligned or too small");
  const int vec = d->dtype == TS_BF16 ? 8 : 4;
  auto rows = [&](const ts_strided& s, int v) {
    return s.ptr && ((uintptr_t)s.ptr & 15u) == 0 && s.sb % v == 0 && s.sh % v == 0 && s.st % v == 0;
  };
  if (!rows(gr->dout, vec) || !rows(gr->dq, 4) || !rows(gr->dk, 4) || !gr->dv.ptr || !gr->dbeta)
    return fail(TS_ERR_VALUE, "delta bwd: missing gradients, or rows that are not aligned");
  if (gr->dout.st < 0 || gr->dout.st >= ((int64_t)1 << 31) / (64 * (16 / vec)))
    return fail(TS_ERR_NOT_IMPLEMENTED, "delta bwd: 64 rows must lie within 2 GiB");
  const int64_t chunks = (int64_t)p.B * p.H * p.nc;
  if (chunks > 0x7fffffff) return fail(TS_ERR_NOT_IMPLEMENTED, "delta bwd: grid too large");
  const size_t es = d->dtype == TS_BF16 ? 2 : 4, dkp = d->dk <= 64 ? 64 : 128;
  const size_t u = (size_t)chunks * p.dvp * 64 * es, s0 = (size_t)chunks * p.dvp * dkp * es;
  p.prep = (float*)saved;
  p.u = (char*)saved + (kept - u - s0);
  p.s0 = (char*)saved + (kept - s0);
  char* ws = (char*)workspace;
  p.dr = ws;
  p.ds = ws + u;
  ws += u + s0;
  if (es == 2) {
    if (!io->low || ((uintptr_t)io->low & 15u))
      return fail(TS_ERR_VALUE, "delta bwd: the low halves' buffer is missing or misaligned");
    p.u_low = ((char*)io->low - (char*)p.u) / 2;
    p.s0_low = ((char*)io->low + u - (char*)p.s0) / 2;
    p.dr_low = p.ds_low = (int64_t)(u + s0) / 2;
    ws += u + s0;
  }
  if (p.nseg > 1) {
    // X of the forward's transfers, which follow its chunks' records
    const size_t states = (size_t)p.B * p.H * p.nseg * p.dvp * dkp * sizeof(float);
    p.seg_x = p.prep + chunks * ts::kRecord;
    p.seg_stride = ts::seg_floats((int)dkp, p.dvp, true);
    p.seg_state = (float*)ws;
    p.seg_n = (float*)(ws + states);
    ws += 2 * states;
  }
  p.dout = gr->dout; p.dval = gr->dv; p.dq = gr->dq; p.dkey = gr->dk;
  p.dbeta = gr->dbeta; p.ddecay = gr->ddecay; p.ddecay_bf16 = p.decay_bf16;
  p.dstate_out = gr->dstate_out; p.dstate = gr->dstate;
  float *gq = nullptr, *gk = nullptr;
  if (p.rep > 1) {
    // per value head in fp32, added up over the heads of a key afterwards
    const int64_t n = (int64_t)p.B * p.H * p.T * p.dk;
    gq = (float*)ws;
    gk = gq + n;
    ws += align16(2 * (size_t)n * sizeof(float));
    const ts_strided f = {gq, (int64_t)p.H * p.T * p.dk, (int64_t)p.T * p.dk, p.dk};
    p.dq = f;
    p.dkey = f;
    p.dkey.ptr = gk;
    p.grad_f32 = 1;
  } else {
    p.grad_f32 = d->dtype == TS_F32;
  }
  if (gr->ddecay_head) {  // one retention a head: its tokens' gradients, then their sum
    p.ddecay = ws;
    p.ddecay_bf16 = 0;
  }
  const bool narrow = d->dk <= 64;
  if (d->dtype == TS_BF16)
    rc = narrow ? backward<ts::bf16, 64>(p, stream) : backward<ts::bf16, 128>(p, stream);
  else
    rc = narrow ? backward<float, 64>(p, stream) : backward<float, 128>(p, stream);
  if (rc) return rc;
  if (p.rep > 1) {
    if (d->dtype == TS_BF16)
      group_sum<ts::bf16>(p, gq, gr->dq, gr->dk, stream);
    else
      group_sum<float>(p, gq, gr->dq, gr->dk, stream);
  }
  if (gr->ddecay_head) {
    if (d->decay_dtype == TS_BF16)
      hipLaunchKernelGGL((ts::delta_head_sum_kernel<ts::bf16>), dim3(p.H), dim3(256), 0, stream, (const float*)p.ddecay,
                         (ts::bf16*)gr->ddecay_head, p.B, p.H, p.T);
    else
      hipLaunchKernelGGL((ts::delta_head_sum_kernel<float>), dim3(p.H), dim3(256), 0, stream, (const float*)p.ddecay,
                         (float*)gr->ddecay_head, p.B, p.H, p.T);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "delta bwd: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}

}  // extern "C"
