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
  float* lse;      // [B,H,T]: log2 of the sum of 2^(scale2 q . k), +inf past a sequence's length
  ts_strided low;  // what rounding leaves of out (bf16), for the backward
  // backward
  ts_strided dout, dq, dk, dv;
  float* delta;  // [B,H,T]: dout . out
  // The keys' gradients in parts: of `owners` heads a batch (the key heads, or where few, the query heads)
  int owners, reps;
  float* rows;  // [B,owners][T][2][d], where owners are the query heads
  float* part;  // [B,owners][chunks + 1][sinks][2][d]: the sinks', near queries', then stretches of the far ones
  int near_tiles, far_tiles, chunks, chunk_tiles;
};

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

// 64 rows of a stream on their way into LDS: 16-byte vectors in registers, at fixed offsets from
// the tile's first row (the host checks that 64 rows lie within 2 GiB).  Rows at or past the
// sequence's length repeat its last one (what they meet is masked); columns past the head's width
// are zero.
template <typename E, int D>
struct WinTile {
  static constexpr int VEC = 16 / (int)sizeof(E), PER = D / VEC, N = TT * PER / 256, STEP = 256 / PER;
  uint4 r[N];
  uint32_t col, pitch;  // bytes
  int row;
  bool on;
  __device__ __forceinline__ void init(int64_t st, int d, int tid) {
    row = tid / PER;
    col = (uint32_t)(tid % PER * 16);
    on = tid % PER * VEC < d;
    pitch = (uint32_t)st * (uint32_t)sizeof(E);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // the tile from row t0 of a sequence at `base` (both uniform)
  __device__ __forceinline__ void fetch(const E* base, int64_t st, int t0, int len) {
    const char* from = (const char*)(base + (int64_t)t0 * st);
    const int last = len - 1 - t0;
    if (!on) return;
    if (last >= TT - 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = *(const uint4*)(from + (size_t)((uint32_t)(row + i * STEP) * pitch + col));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        r[i] = *(const uint4*)(from + (size_t)((uint32_t)min(row + i * STEP, last) * pitch + col));
    }
  }
  __device__ __forceinline__ void store(E* dst) const {
    E* at = dst + row * win_pitch<E, D>() + col / (int)sizeof(E);
#pragma unroll
    for (int i = 0; i < N; ++i) *(uint4*)(at + i * STEP * win_pitch<E, D>()) = r[i];
  }
};

// What a tile of 64 keys from k0 is to the queries q0 .. q1: not seen by any, seen whole by all, or
// cut by their diagonal, by their window's far end (both: that of a short window), or around a sink.
enum WinCut { kWinNone, kWinWhole, kWinDiagonal, kWinEdge, kWinSome };
__device__ __forceinline__ int win_cut(int q0, int q1, int k0, int window, int sinks) {
  const int k1 = k0 + TT - 1;
  if (k0 > q1 || (q0 - k1 >= window && k0 >= sinks)) return kWinNone;
  const bool diagonal = k1 > q0, edge = q1 - k0 >= window && k1 >= sinks;
  if (!diagonal && !edge) return kWinWhole;
  if (edge && (diagonal || k0 < sinks)) return kWinSome;
  return edge ? kWinEdge : kWinDiagonal;
}
// f(kf, e, hidden) for the keys k0 + 16 kf + 4 g + e of a cut tile (a wave-uniform `cut`): whether
// query i does not see them.
template <typename F>
__device__ __forceinline__ void win_mask(int cut, int i, int k0, int g, int window, int sinks, F f) {
  const int a = i - k0 - 4 * g;  // the last key that the query sees, counted as 16 kf + e
  const int b = a - window;      // and the last one before its window
  if (cut == kWinDiagonal) {
#pragma unroll
    for (int j = 0; j < 16; ++j) f(j >> 2, j & 3, 16 * (j >> 2) + (j & 3) > a);
  } else if (cut == kWinEdge) {
#pragma unroll
    for (int j = 0; j < 16; ++j) f(j >> 2, j & 3, 16 * (j >> 2) + (j & 3) <= b);
  } else {
    const int c = min(sinks - k0 - 4 * g, b + 1);  // from here to b: hidden
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int x = 16 * (j >> 2) + (j & 3);
      f(j >> 2, j & 3, (x > a) | ((x <= b) & (x >= c)));
    }
  }
}

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
