// Windowed softmax attention with sinks: what its kernels share (gfx950).
//
// Query i sees key j where j <= i and (i - j < window or j < sinks).
#pragma once

#include "ts_common.h"
#include "ts_tokens.h"

namespace ts {

struct WinP {
  int H, Hkv, rep, T, d;
  int window, sinks;
  float scale, scale2;  // and scale * log2(e)
  ts_strided q, k, v, out;
  const int64_t* lengths;
  float* lse;  // [B,H,T]: log2 of the sum of 2^(scale2 q . k), +inf past a sequence's length
  // backward
  ts_strided dout, dq, dk, dv;
  float* delta;  // [B,H,T]: dout . out
  float* part;   // [B,Hkv][chunks + 1][sinks][2][d]: sums of the sinks' gradients
  int near_tiles, far_tiles, chunks, chunk_tiles;
};

constexpr int kWinQ = 128;  // queries (or keys, backward) of a workgroup, 32 a wave

// 16 bytes of padding keep a tile's rows 4 banks apart.
template <typename E, int D>
constexpr int win_pitch() { return D + 16 / (int)sizeof(E); }

__device__ __forceinline__ int win_length(const WinP& p, int b) {
  if (!p.lengths) return p.T;
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : n > p.T ? p.T : (int)n;
}

__device__ __forceinline__ bool win_hidden(int i, int j, int window, int sinks) {
  return j > i || (i - j >= window && j >= sinks);
}

// Eight consecutive elements of a row, zero past its width and where the row is not one.
__device__ __forceinline__ bf16x8 win_row8(const bf16* row, int col, int d, bool on) {
  uint4 r = make_uint4(0u, 0u, 0u, 0u);
  if (on && col < d) r = *(const uint4*)(row + col);
  return __builtin_bit_cast(bf16x8, r);
}
__device__ __forceinline__ floatx8 win_row8(const float* row, int col, int d, bool on) {
  floatx4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
  if (on && col < d) a = *(const floatx4*)(row + col);
  if (on && col + 4 < d) b = *(const floatx4*)(row + col + 4);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// 64 rows of a stream on their way into LDS: 16-byte vectors in registers, zero past
// the sequence's length and the head's width.
template <typename E, int D>
struct WinTile {
  static constexpr int VEC = 16 / (int)sizeof(E), PER = D / VEC, N = TT * PER / 256;
  uint4 r[N];
  __device__ __forceinline__ void fetch(const E* base, int64_t st, int t0, int len, int d, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * 256, t = t0 + idx / PER, c = idx % PER * VEC;
      r[i] = make_uint4(0u, 0u, 0u, 0u);
      if (t < len && c < d) r[i] = *(const uint4*)(base + (int64_t)t * st + c);
    }
  }
  __device__ __forceinline__ void store(E* dst, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * 256;
      *(uint4*)(dst + idx / PER * win_pitch<E, D>() + idx % PER * VEC) = r[i];
    }
  }
};

// The key tiles (64 keys) that queries q0 .. q1 - 1 see: those of the sinks before the
// window's, then the window's.
struct WinTiles {
  int sink, near0, n;
  __device__ __forceinline__ WinTiles(int q0, int q1, int window, int sinks) {
    near0 = max(0, q0 - window + 1) / TT;
    sink = min((int)(((int64_t)sinks + TT - 1) / TT), near0);
    n = sink + (q1 - 1) / TT - near0 + 1;
  }
  __device__ __forceinline__ int at(int it) const { return (it < sink ? it : near0 + it - sink) * TT; }
};

}  // namespace ts
