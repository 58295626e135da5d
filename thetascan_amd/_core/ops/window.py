"""Windowed softmax attention with sinks: attention whose cost and cache do not grow.

Query i sees key j where ``j <= i`` and ``i - j < window`` or ``j < sinks``: the last
``window`` tokens, its own among them, and the first ``sinks`` ones for good.  It stands
beside the memories (:func:`.scan_hip.linattn`, :func:`.delta.gated_delta_rule`) with their
streams and contract: whole sequences with gradients (ts_window_attention_fwd,
ts_window_attention_bwd), and single tokens against a cache of fixed size
(ts_window_step), a ring of ``window`` slots behind those of the sinks.

bf16 inputs: products take bf16 operands (the probabilities and their gradients rounded
once) and fp32 sums; fp32 inputs compute in fp32.  A value that is not finite reaches the
outputs and gradients alone that its formula has it in.  Where a gradient is recorded, a
call keeps its inputs, its output, a log-sum a query (fp32) and, in bf16, what the output's
rounding left (as large as the output), which the gradients' digits need.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from ... import _lib
from .delta import _on, _rows, _rows_like, _width
from .dispatch import HipOp, refuse_tangents
from .scan_hip import _vec

MAX_HEAD = 128
LEAST_SCALE, MOST_SCALE = 1.2e-38, 2.3e38  # (fp32 holds them, and the latter times log2(e))
_MOST = 2 ** 31 - 1


@functools.lru_cache(maxsize=256)
def _describe(q, kv_heads, dtype, window, sinks, scale) -> _lib.WindowDesc:
    B, H, T, d = q
    return _lib.WindowDesc(B, H, kv_heads, T, _width(dtype, d), _lib.dtype_code(dtype), window, sinks, scale)


@functools.lru_cache(maxsize=256)
def _backward_bytes(q, kv_heads, dtype, window, sinks, scale) -> int:
    n = ctypes.c_size_t()
    desc = _describe(q, kv_heads, dtype, window, sinks, scale)
    _lib.check(_lib.load().ts_window_attention_bwd_workspace_bytes(ctypes.byref(desc), ctypes.byref(n)),
               "ts_window_attention_bwd_workspace_bytes")
    return n.value


def _forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None, window: int, sinks: int,
             scale: float, keep: bool) -> list[torch.Tensor]:
    lib = _lib.load()
    B, H, T, d = q.shape
    vec = _vec(q.dtype)
    desc = _describe(q.shape, k.shape[1], q.dtype, window, sinks, scale)
    (q4, sq), (k4, sk), (v4, sv) = _rows(q, vec), _rows(k, vec), _rows(v, vec)
    out = _rows_like(q, q.dtype, desc.d)
    lse = torch.empty((B, H, T) if keep else 0, dtype=torch.float32, device=q.device)
    low = _rows_like(q, q.dtype, desc.d) if keep and q.dtype == torch.bfloat16 else None
    io = _lib.WindowIO(sq, sk, sv, _lib.strided(out), _lib.ptr(lengths), lse.data_ptr() if keep else None,
                       _lib.strided(low))
    with _on(q.device), _lib.timed("ts_window_attention_fwd", lambda: _lib.nbytes(q4, k4, v4, out)):
        status = lib.ts_window_attention_fwd(ctypes.byref(desc), ctypes.byref(io), _lib.stream_handle(q.device))
    _lib.check(status, "ts_window_attention_fwd")
    return [out if desc.d == d else out[..., :d], lse, q.new_empty(0) if low is None else low]


def _forward_fake(q, k, v, lengths, window, sinks, scale, keep):
    B, H, T, d = q.shape
    out = _rows_like(q, q.dtype, _width(q.dtype, d))[..., :d]
    kept = keep and q.dtype == torch.bfloat16
    return [out, q.new_empty((B, H, T) if keep else (0,), dtype=torch.float32),
            _rows_like(q, q.dtype, _width(q.dtype, d)) if kept else q.new_empty(0)]


def _backward_impl(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                   lse: torch.Tensor, low: torch.Tensor, lengths: torch.Tensor | None, window: int, sinks: int,
                   scale: float) -> list[torch.Tensor]:
    lib = _lib.load()
    d, vec = q.shape[-1], _vec(q.dtype)
    desc = _describe(q.shape, k.shape[1], q.dtype, window, sinks, scale)
    (q4, sq), (k4, sk), (v4, sv), (o4, so) = _rows(q, vec), _rows(k, vec), _rows(v, vec), _rows(out, vec)
    do4, sd = _rows(dout if dout.dtype == q.dtype else dout.to(q.dtype), vec)
    dq, dk, dv = (_rows_like(x, q.dtype, desc.d) for x in (q, k, v))
    io = _lib.WindowIO(sq, sk, sv, so, _lib.ptr(lengths), lse.data_ptr(), _lib.strided(low if low.numel() else None))
    grads = _lib.WindowGrads(sd, _lib.strided(dq), _lib.strided(dk), _lib.strided(dv))
    work = torch.empty(_backward_bytes(q.shape, k.shape[1], q.dtype, window, sinks, scale), dtype=torch.uint8,
                       device=q.device)
    with _on(q.device), _lib.timed("ts_window_attention_bwd", lambda: _lib.nbytes(q4, k4, v4, o4, do4, dq, dk, dv)):
        status = lib.ts_window_attention_bwd(ctypes.byref(desc), ctypes.byref(io), ctypes.byref(grads), work.data_ptr(),
                                             work.numel(), _lib.stream_handle(q.device))
    _lib.check(status, "ts_window_attention_bwd")
    if desc.d != d:
        dq, dk, dv = dq[..., :d], dk[..., :d], dv[..., :d]
    return [dq, dk, dv]


def _backward_fake(dout, q, k, v, out, lse, low, lengths, window, sinks, scale):
    return [_rows_like(x, q.dtype, _width(q.dtype, x.shape[-1]))[..., :x.shape[-1]] for x in (q, k, v)]


def _setup(ctx, inputs, output):
    q, k, v, lengths, ctx.window, ctx.sinks, ctx.scale, _ = inputs
    ctx.save_for_backward(q, k, v, *output, lengths)


def _backward(ctx, grads, bwd):
    if grads[0] is None:
        return (None,) * 8
    q, k, v, out, lse, low, lengths = ctx.saved_tensors
    dq, dk, dv = bwd(grads[0], q, k, v, out, lse, low, lengths, ctx.window, ctx.sinks, ctx.scale)
    return (dq, dk, dv, None, None, None, None, None)


_window_op = HipOp("windowed_attention", forward=_forward, forward_fake=_forward_fake, backward_impl=_backward_impl,
                   backward_fake=_backward_fake, setup=_setup, backward=_backward, once=True)


def _count(what: str, name: str, x, least: int) -> int:
    if isinstance(x, bool) or not isinstance(x, int) or x < least:
        raise ValueError(f"{what}: {name} must be a whole number of at least {least}, got {x!r}")
    return min(x, _MOST)


def _scale(what: str, scale: float | None, d: int) -> float:
    if scale is None:
        return d ** -0.5
    if not LEAST_SCALE <= float(scale) <= MOST_SCALE:
        raise ValueError(f"{what}: scale must be positive, in [{LEAST_SCALE}, {MOST_SCALE}], got {scale}")
    return float(scale)


def _same_place(what: str, q: torch.Tensor, others) -> None:
    device = q.get_device()
    if device < 0:
        raise RuntimeError("hip backend: tensors must live on the GPU (no CPU fallback)")
    for x in others:
        if x is not None and x.get_device() != device:
            if not x.is_cuda:
                raise RuntimeError("hip backend: tensors must live on the GPU (no CPU fallback)")
            raise ValueError(f"{what}: tensors on several devices")


def _heads(what: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.ndim != 4:
            raise ValueError(f"{what}: {name} must be [B,H,T,D], got {tuple(x.shape)}")
    B, H, T, d = q.shape
    Hk = k.shape[1]
    if k.shape != v.shape or k.shape[0] != B or k.shape[2:] != (T, d):
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if min(B, H, Hk, d) < 1 or H % Hk:
        raise ValueError(f"{what}: {H} query heads over {Hk} key heads, {B} sequences, width {d}")
    if d > MAX_HEAD:
        raise NotImplementedError(f"{what}: heads of at most {MAX_HEAD}, got {d}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q, k and v of one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    _lib.dtype_code(q.dtype)


def _sequence_lengths(what: str, lengths: torch.Tensor | None, B: int, name: str = "lengths") -> None:
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"{what}: {name} must be integers [{B}], got {lengths.dtype} {tuple(lengths.shape)}")


def windowed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                       lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Outputs [B,H,T,d] of windowed attention with sinks (module docstring), in the
    query's memory order.

    ``q`` [B,H,T,d], ``k`` and ``v`` [B,Hk,T,d] (bf16 or fp32, any strides, d at most
    128; H a multiple of Hk: query head h reads key head h // (H / Hk)).  ``window``: tokens
    that a query sees back to, its own among them (None: all); ``sinks``: first tokens
    that stay visible.  ``scale`` multiplies the scores (None: d ** -0.5; scores past 2^30 in
    size are not held, and may give NaN).  ``lengths`` [B]
    (integers, on the GPU, clamped to [0, T]) makes a padded batch: tokens at or past a
    sequence's length are not read, give zeros and gradients of zero.

    Differentiable in q, k and v (once, backwards: forward-mode and second derivatives
    are refused).
    """
    what = "windowed_attention"
    _heads(what, q, k, v)
    B, H, T, d = q.shape
    window = _MOST if window is None else _count(what, "window", window, 1)
    sinks = _count(what, "sinks", sinks, 0)
    scale = _scale(what, scale, d)
    _sequence_lengths(what, lengths, B)
    if not torch.compiler.is_compiling():
        refuse_tangents(what, q, k, v)
    _same_place(what, q, (k, v, lengths))
    if T == 0:
        return q.new_empty(B, H, 0, d)
    if lengths is not None:
        lengths = lengths.to(torch.int64).contiguous()
    record = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _window_op(q, k, v, lengths, window, sinks, scale, record)[0]


def _cache(what: str, k: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, sinks: int) -> int:
    """Checks a cache for keys and values like ``k`` and returns its window."""
    B, Hk, _, d = k.shape
    if torch.compiler.is_compiling():
        raise NotImplementedError(f"{what}: a traced call writes into no tensor it is given (the cache)")
    vec = _vec(k.dtype)
    if d % vec:
        raise NotImplementedError(f"{what}: heads in 16-byte vectors, got {d} of {k.dtype}")
    for name, x in (("cache_k", cache_k), ("cache_v", cache_v)):
        if x.ndim != 4 or (x.shape[0], x.shape[1], x.shape[3]) != (B, Hk, d) or x.dtype != k.dtype:
            raise ValueError(f"{what}: {name} must be {k.dtype} [{B},{Hk},slots,{d}], got {x.dtype} {tuple(x.shape)}")
        s = x.stride()
        if s[3] != 1 or (s[0] | s[1] | s[2]) % vec or x.data_ptr() % 16 or any(
                a == 0 and n > 1 for a, n in zip(s, x.shape)):
            raise ValueError(f"{what}: {name} must have contiguous 16-byte rows of its own, got strides {s}")
        if x.requires_grad:
            raise ValueError(f"{what}: {name} takes no part in gradients")
    if cache_k.shape[2] != cache_v.shape[2] or cache_k.shape[2] <= sinks:
        raise ValueError(f"{what}: caches of {cache_k.shape[2]} and {cache_v.shape[2]} slots, {sinks} of them sinks")
    if cache_k.data_ptr() == cache_v.data_ptr():
        raise ValueError(f"{what}: keys and values need a cache each")
    return min(cache_k.shape[2] - sinks, _MOST)


def _meets(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether the stretches of memory that hold two tensors overlap."""
    (a, b), (c, d) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
                      for t in (x, y))
    return a < d and c < b


def _changed(*caches: torch.Tensor) -> None:
    for x in caches:
        if not x.is_inference():
            # (the kernel's writing is autograd's in-place change: what saved the old values says so)
            torch.autograd.graph.increment_version(x)


def _unrecorded(what: str, *tensors: torch.Tensor) -> None:
    refuse_tangents(what, *tensors)
    if torch.is_grad_enabled() and any(x.requires_grad for x in tensors):
        raise ValueError(f"{what}: takes no part in gradients: call it without them")


@functools.lru_cache(maxsize=256)
def _step_plan(q, kv_heads, dtype, window, sinks, scale) -> tuple[_lib.WindowDesc, int]:
    n, desc = ctypes.c_size_t(), _describe(q, kv_heads, dtype, window, sinks, scale)
    _lib.check(_lib.load().ts_window_step_workspace_bytes(ctypes.byref(desc), ctypes.byref(n)),
               "ts_window_step_workspace_bytes")
    return desc, n.value


def windowed_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache_k: torch.Tensor,
                            cache_v: torch.Tensor, positions: torch.Tensor, *, sinks: int = 0,
                            scale: float | None = None) -> torch.Tensor:
    """Outputs [B,H,1,d] of :func:`windowed_attention` for the next token of each
    sequence, whose earlier ones stand in its cache.

    ``q`` [B,H,1,d], ``k`` and ``v`` [B,Hk,1,d] are the new tokens'.  ``cache_k`` and
    ``cache_v`` [B,Hk,sinks + window,d] hold the earlier ones, position n in slot n where n
    is below ``sinks``, else in slot ``sinks + (n - sinks) % window`` (as
    :func:`fill_window_cache` and earlier steps left them); the new key and value are
    written into theirs.  ``positions`` [B] (integers, on the GPU): the new tokens'
    positions, which are the numbers of tokens before them; one below zero marks a free
    place, whose output is zero and whose cache is neither read nor written.  Slots that
    hold no token yet may hold anything.  Without gradients.
    """
    what = "windowed_attention_step"
    _heads(what, q, k, v)
    B, H, T, d = q.shape
    if T != 1:
        raise ValueError(f"{what}: one token of each sequence, got {T}")
    sinks = _count(what, "sinks", sinks, 0)
    window = _cache(what, k, cache_k, cache_v, sinks)
    scale = _scale(what, scale, d)
    _sequence_lengths(what, positions, B, "positions")
    _unrecorded(what, q, k, v)
    _same_place(what, q, (k, v, cache_k, cache_v, positions))
    vec = _vec(q.dtype)
    desc, nbytes = _step_plan(q.shape, k.shape[1], q.dtype, window, sinks, scale)
    (q4, sq), (k4, sk), (v4, sv) = _rows(q, vec), _rows(k, vec), _rows(v, vec)
    positions = positions.to(torch.int64).contiguous()
    out = _rows_like(q, q.dtype, d)
    io = _lib.WindowIO(sq, sk, sv, _lib.strided(out), None, None, _lib.strided(None))
    work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    with _on(q.device), _lib.timed("ts_window_step", lambda: _lib.nbytes(q4, k4, v4, out, cache_k, cache_v)):
        status = _lib.load().ts_window_step(ctypes.byref(desc), ctypes.byref(io), _lib.strided(cache_k),
                                            _lib.strided(cache_v), positions.data_ptr(), _lib.ptr(work), nbytes,
                                            _lib.stream_handle(q.device))
    _lib.check(status, "ts_window_step")
    _changed(cache_k, cache_v)
    return out


def fill_window_cache(k: torch.Tensor, v: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, *,
                      sinks: int = 0, lengths: torch.Tensor | None = None) -> None:
    """Writes a prompt's keys and values [B,Hk,T,d] into caches [B,Hk,sinks + window,d]
    as :func:`windowed_attention_step` takes them: the first ``sinks`` tokens, and the last
    ``window`` ones, of the T or ``lengths`` [B] tokens of each sequence.  Slots that no
    token falls into are left as they are.  Without gradients."""
    what = "fill_window_cache"
    _heads(what, k, k, v)
    B, Hk, T, d = k.shape
    sinks = _count(what, "sinks", sinks, 0)
    window = _cache(what, k, cache_k, cache_v, sinks)
    _sequence_lengths(what, lengths, B)
    _unrecorded(what, k, v)
    _same_place(what, k, (v, cache_k, cache_v, lengths))
    if T == 0:
        return
    # (what stands in a cache itself is read from a copy: slots are written while others are read)
    k, v = (x.clone() if _meets(x, cache_k) or _meets(x, cache_v) else x for x in (k, v))
    vec = _vec(k.dtype)
    desc = _describe(k.shape, Hk, k.dtype, window, sinks, 1.0)
    (k4, sk), (v4, sv) = _rows(k, vec), _rows(v, vec)
    if lengths is not None:
        lengths = lengths.to(torch.int64).contiguous()
    io = _lib.WindowIO(sk, sk, sv, sk, _lib.ptr(lengths), None, _lib.strided(None))
    with _on(k.device), _lib.timed("ts_window_cache_fill", lambda: 2 * _lib.nbytes(k4[:, :, :window + sinks],
                                                                                   v4[:, :, :window + sinks])):
        status = _lib.load().ts_window_cache_fill(ctypes.byref(desc), ctypes.byref(io), _lib.strided(cache_k),
                                                  _lib.strided(cache_v), _lib.stream_handle(k.device))
    _lib.check(status, "ts_window_cache_fill")
    _changed(cache_k, cache_v)
