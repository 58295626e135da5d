// Shared parts of the gated delta rule's kernels (gfx950): chunk layout of the
// workspace and operand helpers.
//
// Mathematics (per batch and value head, state S [dk, dv] fp32):
//   S_t = a_t S_{t-1} + k_t u_t^T,  u_t = b_t (v_t - a_t S_{t-1}^T k_t),  o_t = S_t^T q_t
// For a chunk of 64 tokens with entering state S0 and G_t = sum_{s<=t} log a_s in it:
//   L_ti = b_t e^{G_t - G_i} k_t.k_i  (i < t),   Ti = (I + L)^-1
//   P_ti = e^{G_t - G_i} q_t.k_i      (i <= t)
//   U = Ti b (V - e^G K S0),   O = e^G Q S0 + P U,   S' = e^{G_63} S0 + K^T (e^{G_63 - G} U)
// Every exponent is a difference of sums over a range of tokens: at most zero
// for retentions, and formed in fp64, so a reset (log a = -inf, taken as -1000)
// costs its neighbours no digits.
//
// A token at or past its sequence's length reads as q = k = v = 0, b = 0,
// log a = 0: it writes nothing, and its row and column of Ti are the identity's.
#pragma once

#include "ts_common.h"
#include "ts_tokens.h"

namespace ts {

constexpr int kChunk = 64;
constexpr double kLog2e = 1.4426950408889634074;

// A lower triangular 64 x 64 matrix as MFMA operands: row block r (16 rows)
// and contraction step s (32 columns), the six that hold the triangle.  Lane
// (l16, g) owns row 16r + l16 and columns 32s + 16(j >> 2) + 4g + (j & 3), the
// order in which accumulators of 16-row blocks 2s, 2s+1 hold their rows.
constexpr int kTri = 6;
__device__ __forceinline__ constexpr int tri(int r, int s) { return r < 2 ? r : (r == 2 ? 2 + s : 4 + s); }

// Elements of one fragment set in the workspace.
constexpr int kTriElems = kTri * 64 * 8;

// Parts that a value enters products in: bf16 ones whose sum it is (fp32: itself).  Where
// keys are alike, sums over a chunk cancel, and what one rounding leaves does not.  Three
// hold fp32's 24 bits, for what the state and the outputs come of; two hold 16, for the
// gradients, which are rounded to 8.
template <typename E, int N> constexpr int kParts = sizeof(E) == 2 ? N : 1;

// Per chunk, fp32: the inverse, P, and e^G, e^{G_63 - G}, b (64 each, zero past the
// length) and e^{G_63}.
constexpr int kVec = 3 * kChunk + 4;
constexpr int kRecord = 2 * kTriElems + kVec;

struct DeltaP {
  int B, Hk, H, rep, T, dk, dv, nc;  // nc: chunks of T
  int dvp;                           // dv rounded up to 16
  int beta_bf16, decay_bf16;
  ts_strided q, k, v, beta, decay, out;
  const int64_t* lengths;  // [B] or null
  const float* state;      // [B,H,dk,dv] or null (zero)
  float* state_out;        // or null
  float* prep;             // [B*H*nc] of kRecord
  int nseg, seg_chunks;    // segments of the chain, chunks of each
  float* seg_x;            // [B*H*nseg][seg_stride]: X as rows, N, and (kept) X as columns
  int64_t seg_stride;
  float* seg_state;        // [B*H*nseg][dvp][DK]: states entering the segments (backward:
                           // gradients behind them)
  void* u;                 // kept: [B*H*nc][dvp][64]
  void* s0;                // kept: [B*H*nc][dvp][DK]
  int64_t u_low, s0_low;   // elements from those to what their rounding to bf16 leaves, and from
                           // dr and ds to theirs (fp32: none)
  int64_t dr_low, ds_low;
  // backward
  ts_strided dout, dq, dkey, dval;
  void* dbeta;   // [B,H,T] of beta's dtype
  void* ddecay;  // [B,H,T], decay's dtype (or fp32), or null
  int ddecay_bf16, grad_f32;  // grad_f32: dq and dkey are fp32 (value heads that share keys)
  const float* dstate_out;  // gradient of the final state or null
  float* dstate;            // gradient of the entering state or null
  void* dr;                 // [B*H*nc][dvp][64]
  void* ds;                 // [B*H*nc][dvp][DK]
  float* seg_n;             // [B*H*nseg][dvp][DK]: N of the backward's transfers
  // (of the segments' matrices a wave's accumulators follow one another: block_at)
};

__device__ __forceinline__ int delta_len(const DeltaP& p, int b) {
  if (!p.lengths) return p.T;
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : (n > p.T ? p.T : (int)n);
}
__device__ __forceinline__ float gate_at(const ts_strided& s, int bf, int64_t i) {
  return bf ? tof(((const bf16*)s.ptr)[i]) : ((const float*)s.ptr)[i];
}

template <typename E>
__device__ __forceinline__ typename Frag<E>::f8 zero8() {
  typename Frag<E>::f8 z;
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = (E)0.0f;
  return z;
}
__device__ __forceinline__ floatx4 zero4() { return floatx4{0.f, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ unsigned pack2(float x, float y) {
  typedef float floatx2 __attribute__((ext_vector_type(2)));
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2{x, y}), bf16x2));
}

// Two values' leading bf16 parts, packed, and what they leave.
// (two to a conversion: one at a time takes a conversion each and their packing)
__device__ __forceinline__ unsigned lead2(float& x, float& y) {
  const unsigned h = pack2(x, y);
  x -= __uint_as_float(h << 16);
  y -= __uint_as_float(h & 0xffff0000u);
  return h;
}

// An operand in N parts (fp32: in one), from the accumulators of two 16-row blocks or
// from parts in memory.
template <typename E, int N> struct Parts;
template <int N> struct Parts<bf16, N> {
  bf16x8 p[N];
  __device__ __forceinline__ Parts() {}
  __device__ __forceinline__ Parts(floatx4 a, floatx4 b) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint4 u;
      u.x = lead2(v[0], v[1]);
      u.y = lead2(v[2], v[3]);
      u.z = lead2(v[4], v[5]);
      u.w = lead2(v[6], v[7]);
      p[i] = __builtin_bit_cast(bf16x8, u);
    }
  }
  // The first block's four rows to a, the second's to b, of the second part `low` elements behind.
  __device__ __forceinline__ void store2(bf16* a, bf16* b, int64_t low) const {
    const uint4 h = __builtin_bit_cast(uint4, p[0]), l = __builtin_bit_cast(uint4, p[1]);
    *(uint2*)a = make_uint2(h.x, h.y);
    *(uint2*)b = make_uint2(h.z, h.w);
    *(uint2*)(a + low) = make_uint2(l.x, l.y);
    *(uint2*)(b + low) = make_uint2(l.z, l.w);
  }
};
template <int N> struct Parts<float, N> {
  floatx8 p[1];
  __device__ __forceinline__ Parts() {}
  __device__ __forceinline__ Parts(floatx4 a, floatx4 b) {
    p[0] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  __device__ __forceinline__ void store2(float* a, float* b, int64_t) const {
    *(floatx4*)a = __builtin_shufflevector(p[0], p[0], 0, 1, 2, 3);
    *(floatx4*)b = __builtin_shufflevector(p[0], p[0], 4, 5, 6, 7);
  }
};
// c + x y, the smallest products first; of two operands in parts, those that reach the
// last part's place.
template <typename E, int N>
__device__ __forceinline__ floatx4 mma_parts(typename Frag<E>::f8 x, const Parts<E, N>& y, floatx4 c) {
#pragma unroll
  for (int i = kParts<E, N> - 1; i >= 0; --i) c = mma32(x, y.p[i], c);
  return c;
}
template <typename E, int N>
__device__ __forceinline__ floatx4 mma_parts(const Parts<E, N>& y, typename Frag<E>::f8 x, floatx4 c) {
#pragma unroll
  for (int i = kParts<E, N> - 1; i >= 0; --i) c = mma32(y.p[i], x, c);
  return c;
}
template <typename E, int N>
__device__ __forceinline__ floatx4 mma_parts(const Parts<E, N>& x, const Parts<E, N>& y, floatx4 c) {
#pragma unroll
  for (int sum = kParts<E, N> - 1; sum >= 0; --sum)
#pragma unroll
    for (int i = sum; i >= 0; --i) c = mma32(x.p[i], y.p[sum - i], c);
  return c;
}

// One fragment of a triangular matrix of N parts in LDS, kTriElems from one to the next.
template <int N, typename E>
__device__ __forceinline__ Parts<E, N> get_tri(const E* m, int r, int s, int lane) {
  Parts<E, N> f;
#pragma unroll
  for (int i = 0; i < kParts<E, N>; ++i)
    f.p[i] = *(const typename Frag<E>::f8*)(m + i * kTriElems + (tri(r, s) * 64 + lane) * 8);
  return f;
}
template <int N, typename E>
__device__ __forceinline__ void put_tri(E* m, int r, int s, int lane, const Parts<E, N>& f) {
#pragma unroll
  for (int i = 0; i < kParts<E, N>; ++i)
    *(typename Frag<E>::f8*)(m + i * kTriElems + (tri(r, s) * 64 + lane) * 8) = f.p[i];
}

// Eight columns of an LDS row in accumulator order (32s + 4g.., 32s + 16 + 4g..).
template <typename E>
__device__ __forceinline__ typename Frag<E>::f8 row_perm(const E* row, int s, int g) {
  return LdsIO<E>::cat(LdsIO<E>::ld4(row + 32 * s + 4 * g), LdsIO<E>::ld4(row + 32 * s + 16 + 4 * g));
}

// Operand of the transposed triangle from its LDS copy: row 16r + l16 of Tr^T,
// contraction step s (rows of Tr in accumulator order).
template <typename E> struct TriT;
template <> struct TriT<bf16> {
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
  static __device__ __forceinline__ bf16x8 get(const bf16* t, int r, int s, int lane) {
    const int g = lane >> 4, j = lane & 15;
    const int at = (j & 3) * 128 + (4 * g + (j >> 2)) * 8 + (r & 1) * 4;
    shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(t + tri(2 * s + 1, r >> 1) * 512 + at));
    shortx4 lo = {0, 0, 0, 0};
    // (row block 2s of step s is past the triangle for the odd block beside it)
    if (2 * s >= r) lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(t + tri(2 * s, r >> 1) * 512 + at));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};
template <> struct TriT<float> {
  static __device__ __forceinline__ floatx8 get(const float* t, int r, int s, int lane) {
    const int g = lane >> 4, l16 = lane & 15;
    floatx8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int rb = 2 * s + (e >> 2);  // row block of Tr
      const int at = (l16 >> 2) * 128 + (4 * g + (e & 3)) * 8 + (r & 1) * 4 + (l16 & 3);
      v[e] = rb >= r ? t[tri(rb, r >> 1) * 512 + at] : 0.f;
    }
    return v;
  }
};

// The same of a matrix in N parts.
template <int N, typename E>
__device__ __forceinline__ Parts<E, N> get_tri_t(const E* t, int r, int s, int lane) {
  Parts<E, N> f;
#pragma unroll
  for (int i = 0; i < kParts<E, N>; ++i) f.p[i] = TriT<E>::get(t + i * kTriElems, r, s, lane);
  return f;
}

// A [64 x W] token tile on its way from global memory to LDS rows: vector idx =
// tid + i * THREADS.  Columns at or past `width` (a multiple of a vector) are
// zero.  Loads have no branches, so that the wait for them is counted: rows at or
// past `len` read the last row instead, and what is made of them meets zeros (b,
// e^G and e^{G_63 - G}, and the rows of the triangles, of tokens past the length).
template <typename E, int W, int THREADS>
struct ChunkTile {
  static constexpr int VEC = 16 / (int)sizeof(E);
  static constexpr int PER = W / VEC;
  static constexpr int SLOTS = kChunk * PER / THREADS;
  uint4 r[SLOTS];
  unsigned off[SLOTS];  // bytes from the chunk's first row (the host checks that they fit)
  unsigned col[SLOTS];  // those of its column
  unsigned row_bytes;
  bool narrow;
  __device__ __forceinline__ void init(int64_t st, int width, int tid) {
    row_bytes = (unsigned)(st * (int)sizeof(E));
    narrow = width < W;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int idx = tid + i * THREADS, c = (idx % PER) * VEC;
      col[i] = c < width ? c * (unsigned)sizeof(E) : 0u;
      off[i] = (unsigned)(idx / PER) * row_bytes + col[i];
    }
  }
  __device__ __forceinline__ void fetch(const E* base, int64_t st, int t0, int len) {
    const char* first = (const char*)(base + (int64_t)t0 * st);
    const unsigned last = (unsigned)(min(len - t0, kChunk) - 1) * row_bytes;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) r[i] = *(const uint4*)(first + min(off[i], last + col[i]));
  }
  __device__ __forceinline__ void store(E* dst, int pitch, int width, int tid) {
    if (narrow) {  // uniform
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        if (((tid + i * THREADS) % PER) * VEC >= width) r[i] = make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int idx = tid + i * THREADS;
      *(uint4*)(dst + (idx / PER) * pitch + (idx % PER) * VEC) = r[i];
    }
  }
  // Rows at or past the length zeroed (a kernel that takes its tile on its own).
  __device__ __forceinline__ void clear(int t0, int len, int tid) {
    if (t0 + kChunk <= len) return;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (t0 + (tid + i * THREADS) / PER >= len) r[i] = make_uint4(0u, 0u, 0u, 0u);
  }
};

// A triangular matrix of a chunk's record on its way to LDS, where it stands in N parts.
template <int N>
struct TriTile {
  static constexpr int SLOTS = kTriElems / 4 / 256;
  static_assert(SLOTS * 4 * 256 == kTriElems, "whole slots of 256 threads");
  floatx4 r[SLOTS];
  __device__ __forceinline__ void fetch(const float* src, int tid) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) r[i] = ((const floatx4*)src)[tid + i * 256];
  }
  __device__ __forceinline__ void store(float* dst, int tid) const {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) ((floatx4*)dst)[tid + i * 256] = r[i];
  }
  __device__ __forceinline__ void store(bf16* dst, int tid) const {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      float x = r[i][0], y = r[i][1], z = r[i][2], w = r[i][3];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const unsigned a = lead2(x, y), b = lead2(z, w);
        ((uint2*)(dst + k * kTriElems))[tid + i * 256] = make_uint2(a, b);
      }
    }
  }
};

// Waves a SIMD to compile for: two workgroups a CU, or one where its chunk alone fills
// the LDS (fp32 and 128 keys; compiled for two, its registers spill: 32 heads of 2048 x 128
// forward 281 us against 230, backward 657 against 417).
template <typename E, int DK> constexpr int kWaves = DK == 128 && sizeof(E) == 4 ? 1 : 2;

// Whether a value is NaN or infinite, gathered over several: NaN then, zero otherwise.
__device__ __forceinline__ float taint(float x, float sofar) { return fmaf(x, 0.f, sofar); }

// Every load so far has landed (counted from here, a loop's waits are for its own).
__device__ __forceinline__ void loads_landed() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// Four consecutive rows of column c0 + l16 of an LDS tile, from row r0 + 4g.
template <typename E>
__device__ __forceinline__ floatx4 col4(const E* rows, int pitch, int r0, int c0, int lane);
template <>
__device__ __forceinline__ floatx4 col4<bf16>(const bf16* rows, int pitch, int r0, int c0, int lane) {
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
  const int g = lane >> 4, j = lane & 15;
  const bf16* a = rows + (r0 + 4 * g + (j >> 2)) * pitch + c0 + 4 * (j & 3);
  const bf16x4 v = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)a));
  return floatx4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
template <>
__device__ __forceinline__ floatx4 col4<float>(const float* rows, int pitch, int r0, int c0, int lane) {
  const float* a = rows + (r0 + 4 * (lane >> 4)) * pitch + c0 + (lane & 15);
  return floatx4{a[0], a[pitch], a[2 * pitch], a[3 * pitch]};
}

// Where a lane's part of the 16 x 16 block (rows 16d.., columns 16cb..) of a [DK x W]
// fp32 matrix stands: blocks of a column block follow one another, in a block the
// lanes' accumulators.
template <int DK>
__device__ __forceinline__ int block_at(int cb, int d, int lane) { return ((cb * (DK / 16) + d) * 64 + lane) * 4; }
// Floats of a segment's transfer.
inline int64_t seg_floats(int dkp, int dvp, bool kept) { return (int64_t)(dkp * (kept ? 2 : 1) + dvp) * dkp; }

template <int DK, bool BACK>
__global__ void delta_segments_kernel(DeltaP p);

int delta_segments(const ts_delta_desc* d);
int delta_check(const ts_delta_desc* d, const ts_delta_io* io, DeltaP* p, const char* what);

}  // namespace ts
