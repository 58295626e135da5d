// One token of each sequence against its ring cache: windowed softmax attention with sinks
// for serving (gfx950).
//
// The token of position n stands in slot n where n < sinks, else in slot
// sinks + (n - sinks) % window, so every slot that holds a token is visible to the newest,
// and the softmax over them does not care for their order.  Bound by the cache's bytes (64 sequences of 8
// 128-wide key heads, 4096 slots: 148 us, 5.0 TB/s), a single sequence by its two launches (5 us, and 12
// of the join).
//
// The query heads that share a key head are the columns of the products (16 at a time), so
// a key is read once for all of them.  A wave takes 32 slots at a time: keys straight from
// memory as the rows of S^T = K Q^T, values through its own LDS rows, which
// O^T += V^T P^T reads by columns; no barrier in the loop.  A group's slots are spread over
// the waves of a workgroup and, where groups are few, over several workgroups, whose sums
// a second kernel joins.  The new key and value are taken from the call where their slot is
// read, and written there by one workgroup of the group.

#include "ts_window.h"

#include <string.h>

namespace ts {

int window_setup(const ts_window_desc* d, const ts_window_io* io, WinP* p);

struct WinStepP {
  int H, Hkv, rep, d, window, sinks, splits;
  float scale2;
  ts_strided q, k, v, out, ck, cv;
  const int64_t* positions;
  float* part;   // [B * H][splits][d]
  float2* sums;  // [B * H][splits]: maximum and sum
};

constexpr int kStepSlots = 32;  // slots of a wave at a time

__device__ __forceinline__ int step_slots(int64_t pos, int window, int sinks) {
  const int64_t n = (int64_t)sinks + window;
  return pos + 1 < n ? (int)(pos + 1) : (int)n;
}
__device__ __forceinline__ int step_slot(int64_t pos, int window, int sinks) {
  return pos < sinks ? (int)pos : sinks + (int)((pos - sinks) % window);
}

template <typename E, int D>
__global__ __launch_bounds__(256) void window_step_kernel(WinStepP p) {
  typedef LdsIO<E> IO;
  typedef TokFrag<E> TF;
  typedef typename Frag<E>::f8 f8;
  constexpr int P = win_pitch<E, D>(), DB = D / 16, KB = D / 32, VEC = 16 / (int)sizeof(E), PER = D / VEC;
  constexpr int NV = kStepSlots * PER / 64;
  extern __shared__ __align__(16) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
  E* vt = (E*)lds + w * kStepSlots * P;
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv, z = blockIdx.z * 16, d = p.d;
  const int heads = min(16, p.rep - z), h0 = hk * p.rep + z;
  const int64_t pos = p.positions[b];
  if (pos < 0) {  // a free place (uniform)
    if (blockIdx.y == 0)
      for (int i = tid; i < heads * d; i += 256)
        ((E*)p.out.ptr)[b * p.out.sb + (h0 + i / d) * p.out.sh + i % d] = cvt<E>(0.f);
    return;
  }
  const int n = step_slots(pos, p.window, p.sinks), mine = step_slot(pos, p.window, p.sinks);
  const E* kb = (const E*)p.ck.ptr + b * p.ck.sb + hk * p.ck.sh;
  const E* vb = (const E*)p.cv.ptr + b * p.cv.sb + hk * p.cv.sh;
  const E* kn = (const E*)p.k.ptr + b * p.k.sb + hk * p.k.sh;
  const E* vn = (const E*)p.v.ptr + b * p.v.sb + hk * p.v.sh;
  if (blockIdx.y == 0 && z == 0) {
    for (int i = tid; i < 2 * (d / VEC); i += 256) {
      const int c = i % (d / VEC) * VEC;
      if (i < d / VEC)
        *(uint4*)((E*)p.ck.ptr + b * p.ck.sb + hk * p.ck.sh + (int64_t)mine * p.ck.st + c) = *(const uint4*)(kn + c);
      else
        *(uint4*)((E*)p.cv.ptr + b * p.cv.sb + hk * p.cv.sh + (int64_t)mine * p.cv.st + c) = *(const uint4*)(vn + c);
    }
  }
  f8 qf[KB];
  {
    const E* row = (const E*)p.q.ptr + b * p.q.sb + (h0 + min(l16, heads - 1)) * p.q.sh;
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) qf[kk] = win_row8(row, 32 * kk + 8 * g, d, l16 < heads);
  }
  floatx4 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
  float mx = -INFINITY, sum = 0.f;

  const int tiles = (n + kStepSlots - 1) / kStepSlots, per = (tiles + p.splits - 1) / p.splits;
  const int end = min(tiles, ((int)blockIdx.y + 1) * per);
  for (int it = (int)blockIdx.y * per + w; it < end; it += 4) {
    const int s0 = it * kStepSlots;
    f8 kr[2][KB];
    uint4 vr[NV];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int slot = s0 + 16 * f + l16;
      const E* row = slot == mine ? kn : kb + (int64_t)slot * p.ck.st;
#pragma unroll
      for (int kk = 0; kk < KB; ++kk) kr[f][kk] = win_row8(row, 32 * kk + 8 * g, d, slot < n);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = lane + i * 64, slot = s0 + idx / PER, c = idx % PER * VEC;
      const E* row = slot == mine ? vn : vb + (int64_t)slot * p.cv.st;
      vr[i] = make_uint4(0u, 0u, 0u, 0u);
      if (slot < n && c < d) vr[i] = *(const uint4*)(row + c);
    }
    floatx4 s[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      s[f] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KB; ++kk) s[f] = mma32(kr[f][kk], qf[kk], s[f]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + 16 * f + 4 * g + i >= n) s[f][i] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = fmaxf(m, s[f][i]);
    m = fmaxf(mx, max_g(m));
    const float top = m == -INFINITY ? 0.f : m;
    const float fac = __builtin_amdgcn_exp2f((mx - top) * p.scale2), c = top * p.scale2;
    mx = m;
    float part = 0.f;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[f][i] = __builtin_amdgcn_exp2f(fmaf(s[f][i], p.scale2, -c));
        part += s[f][i];
      }
    sum = fmaf(sum, fac, part);
    wave_lds_sync();  // the last tile's columns are read
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = lane + i * 64;
      *(uint4*)(vt + idx / PER * P + idx % PER * VEC) = vr[i];
    }
    wave_lds_sync();
    const f8 pf = IO::from_acc(s[0], s[1]);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[db][i] *= fac;
      o[db] = mma32(TF::get(vt, P, db * 16, 0, lane), pf, o[db]);
    }
  }
  sum = sum_g(sum);
  // the waves' sums: rows of D floats a head, behind them the maxima and sums
  __syncthreads();
  float* ws = (float*)lds;
  float2* ms = (float2*)(ws + 4 * 16 * (D + 4));
  if (g == 0) ms[w * 16 + l16] = make_float2(mx, sum);
#pragma unroll
  for (int db = 0; db < DB; ++db) *(floatx4*)(ws + (w * 16 + l16) * (D + 4) + db * 16 + 4 * g) = o[db];
  __syncthreads();
  for (int i = tid; i < heads * d; i += 256) {
    const int hq = i / d, c = i % d;
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u) m = fmaxf(m, ms[u * 16 + hq].x);
    const float top = m == -INFINITY ? 0.f : m;
    float total = 0.f, x = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float2 one = ms[u * 16 + hq];
      const float f = __builtin_amdgcn_exp2f((one.x - top) * p.scale2);
      total = fmaf(one.y, f, total);
      x = fmaf(ws[(u * 16 + hq) * (D + 4) + c], f, x);
    }
    const int64_t bh = (int64_t)b * p.H + h0 + hq;
    if (p.splits == 1) {
      ((E*)p.out.ptr)[b * p.out.sb + (h0 + hq) * p.out.sh + c] = cvt<E>(x / total);
    } else {
      p.part[(bh * p.splits + blockIdx.y) * d + c] = x;
      if (c == 0) p.sums[bh * p.splits + blockIdx.y] = make_float2(m, total);
    }
  }
}

template <typename E>
__global__ __launch_bounds__(128) void window_join_kernel(WinStepP p) {
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H, c = threadIdx.x;
  if (c >= p.d || p.positions[b] < 0) return;
  const float2* sums = p.sums + (int64_t)blockIdx.x * p.splits;
  const float* part = p.part + (int64_t)blockIdx.x * p.splits * p.d + c;
  float m = -INFINITY;
  for (int i = 0; i < p.splits; ++i) m = fmaxf(m, sums[i].x);
  const float top = m == -INFINITY ? 0.f : m;
  float total = 0.f, x = 0.f;
  for (int i = 0; i < p.splits; ++i) {
    const float f = __builtin_amdgcn_exp2f((sums[i].x - top) * p.scale2);
    total = fmaf(sums[i].y, f, total);
    x = fmaf(part[(int64_t)i * p.d], f, x);
  }
  ((E*)p.out.ptr)[b * p.out.sb + h * p.out.sh + c] = cvt<E>(x / total);
}

struct WinFillP {
  int Hkv, T, d, window, sinks;
  ts_strided k, v, ck, cv;
  const int64_t* lengths;
};

// A 16-byte vector of a slot a thread, for the keys (blockIdx.z 0) or the values.
template <typename E>
__global__ __launch_bounds__(256) void window_fill_kernel(WinFillP p) {
  constexpr int VEC = 16 / (int)sizeof(E);
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv, per = p.d / VEC;
  const int64_t at = (int64_t)blockIdx.y * 256 + threadIdx.x;
  const int64_t slot = at / per, c = at % per * VEC;
  int64_t len = p.lengths ? p.lengths[b] : p.T;
  if (len > p.T) len = p.T;
  if (slot >= (int64_t)p.sinks + p.window || slot >= len) return;
  // the newest token of this slot
  const int64_t t = slot < p.sinks ? slot : slot + (len - 1 - slot) / p.window * p.window;
  const ts_strided& from = blockIdx.z ? p.v : p.k;
  const ts_strided& to = blockIdx.z ? p.cv : p.ck;
  *(uint4*)((E*)to.ptr + b * to.sb + hk * to.sh + slot * to.st + c) =
      *(const uint4*)((const E*)from.ptr + b * from.sb + hk * from.sh + t * from.st + c);
}

}  // namespace ts

namespace {

using ts::fail;
using ts::WinStepP;

bool rows16(const ts_strided& s, int vec) {
  return s.ptr && ((uintptr_t)s.ptr & 15u) == 0 && s.sb % vec == 0 && s.sh % vec == 0 && s.st % vec == 0;
}

// Sequences and heads, widths and the ring; T plays no part.
int step_setup(const ts_window_desc* d) {
  if (!d) return fail(TS_ERR_VALUE, "window step: no description");
  ts_window_desc one = *d;
  one.T = 1;
  ts::WinP p;
  const int rc = ts::window_setup(&one, nullptr, &p);
  if (rc) return rc;
  if ((int64_t)d->sinks + d->window > 0x7fffffff - 64)
    return fail(TS_ERR_NOT_IMPLEMENTED, "window step: too many slots");
  return TS_OK;
}

// Workgroups a group of heads: some 1024 in all, of 32 slots a wave at least (us for some 256, 512, 1024 and 2048:
// one sequence of 4 key heads and 4096 slots 17 each, eight 16, 17, 23, 22, 64 of 8 98 each: the join of
// many parts costs what the reading gains).
int step_splits(const ts_window_desc* d) {
  const int64_t groups = (int64_t)d->B * d->Hkv * ((d->H / d->Hkv + 15) / 16);
  const int64_t most = ((int64_t)d->sinks + d->window + 4 * ts::kStepSlots - 1) / (4 * ts::kStepSlots);
  const int64_t want = 1024 / groups;
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

template <typename E, int D>
int step(const WinStepP& p, int B, hipStream_t stream) {
  const int tiles = 4 * ts::kStepSlots * ts::win_pitch<E, D>() * (int)sizeof(E);
  const int sums = 4 * 16 * (D + 4) * 4 + 4 * 16 * 8;
  const int lds = tiles > sums ? tiles : sums;
  hipError_t e = ts::ensure_lds_limit((const void*)ts::window_step_kernel<E, D>, lds);
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window step: %s", hipGetErrorString(e));
  const dim3 grid((unsigned)(B * p.Hkv), (unsigned)p.splits, (unsigned)((p.rep + 15) / 16));
  hipLaunchKernelGGL((ts::window_step_kernel<E, D>), grid, dim3(256), lds, stream, p);
  if (p.splits > 1)
    hipLaunchKernelGGL((ts::window_join_kernel<E>), dim3((unsigned)(B * p.H)), dim3(128), 0, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window step: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}

}  // namespace

extern "C" {

int ts_window_step_workspace_bytes(const ts_window_desc* d, size_t* bytes) {
  const int rc = step_setup(d);
  if (rc) return rc;
  const int splits = step_splits(d);
  if (bytes) *bytes = splits == 1 ? 0 : (size_t)d->B * d->H * splits * ((size_t)d->d + 2) * 4;
  return TS_OK;
}

int ts_window_step(const ts_window_desc* d, const ts_window_io* io, ts_strided ck, ts_strided cv,
                   const int64_t* positions, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const int rc = step_setup(d);
  if (rc) return rc;
  const int vec = d->dtype == TS_BF16 ? 8 : 4;
  if (!io || !positions) return fail(TS_ERR_VALUE, "window step: missing tensors");
  for (const ts_strided* s : {&io->q, &io->k, &io->v, &io->out, (const ts_strided*)&ck, (const ts_strided*)&cv})
    if (!rows16(*s, vec)) return fail(TS_ERR_VALUE, "window step: rows must be 16-byte aligned");
  WinStepP p;
  memset(&p, 0, sizeof(p));
  p.H = d->H; p.Hkv = d->Hkv; p.rep = d->H / d->Hkv; p.d = d->d; p.window = d->window; p.sinks = d->sinks;
  p.splits = step_splits(d);
  p.scale2 = d->scale * 1.44269504088896340736f;
  p.q = io->q; p.k = io->k; p.v = io->v; p.out = io->out; p.ck = ck; p.cv = cv;
  p.positions = positions;
  if (p.splits > 1) {
    const size_t need = (size_t)d->B * d->H * p.splits * ((size_t)d->d + 2) * 4;
    if (!workspace || ((uintptr_t)workspace & 15u) || workspace_bytes < need)
      return fail(TS_ERR_VALUE, "window step: workspace of %zu bytes, 16-byte aligned", need);
    p.part = (float*)workspace;
    p.sums = (float2*)(p.part + (size_t)d->B * d->H * p.splits * d->d);
  }
  if (d->dtype == TS_BF16)
    return d->d <= 64 ? step<ts::bf16, 64>(p, d->B, stream) : step<ts::bf16, 128>(p, d->B, stream);
  return d->d <= 64 ? step<float, 64>(p, d->B, stream) : step<float, 128>(p, d->B, stream);
}

int ts_window_cache_fill(const ts_window_desc* d, const ts_window_io* io, ts_strided ck, ts_strided cv,
                         hipStream_t stream) {
  const int rc = step_setup(d);
  if (rc) return rc;
  if (d->T < 0) return fail(TS_ERR_VALUE, "window cache: bad length");
  if (d->T == 0) return TS_OK;
  const int vec = d->dtype == TS_BF16 ? 8 : 4;
  if (!io) return fail(TS_ERR_VALUE, "window cache: missing tensors");
  for (const ts_strided* s : {&io->k, &io->v, (const ts_strided*)&ck, (const ts_strided*)&cv})
    if (!rows16(*s, vec)) return fail(TS_ERR_VALUE, "window cache: rows must be 16-byte aligned");
  ts::WinFillP p;
  memset(&p, 0, sizeof(p));
  p.Hkv = d->Hkv; p.T = d->T; p.d = d->d; p.window = d->window; p.sinks = d->sinks;
  p.k = io->k; p.v = io->v; p.ck = ck; p.cv = cv; p.lengths = io->lengths;
  // (slots that a prompt this long reaches)
  int64_t slots = (int64_t)d->sinks + d->window;
  if (slots > d->T) slots = d->T;
  const int64_t blocks = (slots * (d->d / vec) + 255) / 256;
  if (blocks > 65535) return fail(TS_ERR_NOT_IMPLEMENTED, "window cache: too many slots");
  const dim3 grid((unsigned)(d->B * (int64_t)d->Hkv), (unsigned)blocks, 2);
  if (d->dtype == TS_BF16)
    hipLaunchKernelGGL((ts::window_fill_kernel<ts::bf16>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((ts::window_fill_kernel<float>), grid, dim3(256), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TS_ERR_RUNTIME, "window cache: launch failed: %s", hipGetErrorString(e));
  return TS_OK;
}

}  // extern "C"
