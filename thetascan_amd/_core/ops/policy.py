"""The clipped policy loss with a KL term, on (soft-capped) logits.

What follows rollouts where the soft-capped cross entropy
(:func:`.rowglue.softcap_cross_entropy`) follows plain text: per row n of the
logits, with ``y = cap tanh(z / cap)`` (or z), ``lp = log softmax(y)[token]`` and
``r = exp(lp - old)``::

    loss = sum_n w_n [ -min(r A, clip(r, 1 - low, 1 + high) A)
                       + kl (exp(ref - lp) - (ref - lp) - 1) ]

One pass over the logits a direction (ts_policy_loss_fwd, ts_policy_loss_bwd);
where a gradient is recorded and rows are long (and not few), the forward gives the gradient for a
unit upstream gradient too, which the backward forms again where it is another (as does a
second backward of the same loss).  It is as large as the logits and held from the
forward to the backward, as a saved tensor: offloading hooks and (non-reentrant)
activation checkpointing see it.  A loss whose value alone is wanted is called
without gradients.  Neither the capped logits nor the
probabilities are stored.  A row of weight zero
(a prompt's, a padding's) is not read.
"""
from __future__ import annotations

import ctypes
import functools
import threading

import torch

from ... import _lib
from .delta import _on
from .dispatch import HipOp, eager_forward, refuse_tangents

_GRADIENT = threading.local()  # the gradient that an eager forward leaves for its setup


@functools.lru_cache(maxsize=256)
def _describe(rows, stride, V, dtype, cap, kl, low, high) -> _lib.PolicyDesc:
    return _lib.PolicyDesc(rows, stride if rows > 1 else V, V, _lib.dtype_code(dtype), cap, 0, kl, low, high)


def _desc(z: torch.Tensor, cap: float, kl: float = 0.0, low: float = 0.0, high: float = 0.0) -> _lib.PolicyDesc:
    rows, V = z.shape
    return _describe(rows, z.stride(0), V, z.dtype, cap, kl, low, high)


@functools.lru_cache(maxsize=256)
def _plan(rows: int, V: int, dtype: int, cap: bool) -> tuple[int, bool]:
    """Partial sums of a call, and whether one pass gives the gradient too."""
    lib, n, one = _lib.load(), ctypes.c_int64(), ctypes.c_int32()
    desc = _lib.PolicyDesc(rows, V, V, dtype, 1.0 if cap else 0.0, 0, 0.0, 0.0, 0.0)
    _lib.check(lib.ts_policy_loss_parts(ctypes.byref(desc), ctypes.byref(n)), "ts_policy_loss_parts")
    _lib.check(lib.ts_policy_one_pass(ctypes.byref(desc), ctypes.byref(one)), "ts_policy_one_pass")
    return n.value, bool(one.value)


def _capture(device: torch.device) -> int:
    """The graph that the device's current stream is captured into (0: none)."""
    if not torch.cuda.is_current_stream_capturing():
        return 0
    n = ctypes.c_uint64()
    _lib.check(_lib.load().ts_capture_id(_lib.stream_handle(device), ctypes.byref(n)), "ts_capture_id")
    return n.value


def _rows(z: torch.Tensor) -> torch.Tensor:
    """Logits [rows, V] with contiguous rows (any distance apart)."""
    return z if z.stride(1) == 1 or z.shape[1] == 1 else z.contiguous()


def _forward(z: torch.Tensor, tokens: torch.Tensor, old: torch.Tensor, adv: torch.Tensor, ref: torch.Tensor | None,
             weights: torch.Tensor | None, low: float, high: float, kl: float, cap: float) -> list[torch.Tensor]:
    lib = _lib.load()
    z = _rows(z)
    rows = z.shape[0]
    desc = _desc(z, cap, kl, low, high)
    parts, one_pass = _plan(rows, z.shape[1], desc.dtype, cap > 0.0)
    loss = torch.empty((), dtype=torch.float32, device=z.device)
    lp = torch.empty(rows, dtype=torch.float32, device=z.device)
    # dloss/dlp, the maximum and the logarithm of the sum of each row; the parts of the loss (fp64) before them
    saved = torch.empty(max(2 * parts + 3 * rows, 2), dtype=torch.float32, device=z.device)
    at = saved.data_ptr()
    coef = at + 8 * parts
    dz = None
    if one_pass and rows and eager_forward():
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    io = _lib.PolicyIO(z.data_ptr(), tokens.data_ptr(), old.data_ptr(), _lib.ptr(ref), adv.data_ptr(),
                       _lib.ptr(weights), lp.data_ptr(), coef, coef + 4 * rows, at, loss.data_ptr(), _lib.ptr(dz))
    with _on(z.device), _lib.timed("ts_policy_loss_fwd", lambda: _lib.nbytes(z, tokens, old, adv, ref, weights, lp, dz)):
        status = lib.ts_policy_loss_fwd(ctypes.byref(desc), ctypes.byref(io), _lib.stream_handle(z.device))
        graph = 0 if dz is None else _capture(z.device)
    _lib.check(status, "ts_policy_loss_fwd")
    if dz is not None:
        _GRADIENT.of = (loss, dz, graph)
    return [loss, lp, saved]


def _forward_fake(z, tokens, old, adv, ref, weights, low, high, kl, cap):
    # (a traced size becomes a number here: the parts follow no formula of it)
    parts = _plan(int(z.shape[0]), int(z.shape[1]), _lib.dtype_code(z.dtype), cap > 0.0)[0]
    return [z.new_empty((), dtype=torch.float32), z.new_empty(z.shape[0], dtype=torch.float32),
            z.new_empty(max(2 * parts + 3 * z.shape[0], 2), dtype=torch.float32)]


def _backward_impl(g: torch.Tensor, z: torch.Tensor, tokens: torch.Tensor, weights: torch.Tensor | None,
                   saved: torch.Tensor, cap: float) -> torch.Tensor:
    return _gradient(g, z, tokens, weights, saved, cap, None)


def _gradient(g, z, tokens, weights, saved, cap, formed: torch.Tensor | None) -> torch.Tensor:
    """The logits' gradient; ``formed`` is the forward's, for a unit ``g``, which
    becomes it."""
    lib = _lib.load()
    z = _rows(z)
    rows = z.shape[0]
    dz = torch.empty(z.shape, dtype=z.dtype, device=z.device) if formed is None else formed
    g32 = g if g.dtype == torch.float32 else g.to(torch.float32)
    coef = saved.data_ptr() + 4 * (saved.numel() - 3 * rows)
    io = _lib.PolicyIO(z.data_ptr(), tokens.data_ptr(), None, None, None, _lib.ptr(weights), None, coef,
                       coef + 4 * rows, None, None, dz.data_ptr())
    desc, name = _desc(z, cap), "ts_policy_loss_bwd" if formed is None else "ts_policy_loss_scale"
    with _on(z.device), _lib.timed(name, lambda: _lib.nbytes(z, tokens, dz)):
        stream = _lib.stream_handle(z.device)
        if formed is None:
            status = lib.ts_policy_loss_bwd(ctypes.byref(desc), ctypes.byref(io), g32.data_ptr(), dz.data_ptr(), stream)
        else:
            status = lib.ts_policy_loss_scale(ctypes.byref(desc), ctypes.byref(io), g32.data_ptr(), stream)
    _lib.check(status, name)
    return dz


def _backward_fake(g, z, tokens, weights, saved, cap):
    return z.new_empty(z.shape)


def _setup(ctx, inputs, output):
    z, tokens, weights, ctx.cap = inputs[0], inputs[1], inputs[5], inputs[9]
    left, _GRADIENT.of = getattr(_GRADIENT, "of", None), None
    dz, ctx.graph = left[1:] if left is not None and left[0] is output[0] else (None, None)
    ctx.save_for_backward(z, tokens, weights, output[2], dz)


def _backward(ctx, grads, bwd):
    if grads[0] is None:
        return (None,) * 10
    z, tokens, weights, saved, dz = ctx.saved_tensors
    graph, ctx.graph = ctx.graph, None
    if dz is not None and graph is not None:
        # (a backward in a graph of its own may be replayed more often than the
        # forward, and would take another gradient's for the unit one's; each is handed out once)
        with _on(dz.device):
            same = _capture(dz.device) == graph
        if same:
            # (.data: what the caller does with it is no change of the saved tensor)
            return (_gradient(grads[0], z, tokens, weights, saved, ctx.cap, dz.data), *(None,) * 9)
    return (bwd(grads[0], z, tokens, weights, saved, ctx.cap), *(None,) * 9)


_policy_op = HipOp("policy_loss", forward=_forward, forward_fake=_forward_fake, backward_impl=_backward_impl,
                   backward_fake=_backward_fake, setup=_setup, backward=_backward, once=True)


def _row_values(x: torch.Tensor | None) -> torch.Tensor | None:
    """One fp32 value a row, contiguous, without its gradient."""
    if x is None or (x.dtype == torch.float32 and x.ndim == 1 and not x.requires_grad and x.is_contiguous()):
        return x
    return x.detach().to(torch.float32).reshape(-1).contiguous()


def _flat(what: str, logits: torch.Tensor, tokens: torch.Tensor, softcap: float | None,
          rows: dict) -> tuple[torch.Tensor, torch.Tensor, float, dict]:
    """The logits as [rows, V], the tokens and per-row tensors (fp32) as [rows]."""
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [..., V], got {tuple(logits.shape)}")
    shape = logits.shape[:-1]
    if tokens.shape != shape or tokens.dtype != torch.int64:
        raise ValueError(f"{what}: tokens must be int64 {tuple(shape)}, got {tokens.dtype} {tuple(tokens.shape)}")
    for name, x in rows.items():
        if x is not None and (x.shape != shape or not (x.is_floating_point() or name == "weights")):
            raise ValueError(f"{what}: {name} must be floating-point {tuple(shape)}, got {x.dtype} {tuple(x.shape)}")
    cap = 0.0 if softcap is None else float(softcap)
    if softcap is not None and not 1e-29 <= cap <= 1e29:
        raise ValueError(f"{what}: softcap must be positive, in [1e-29, 1e29] (None: no cap), got {softcap}")
    _lib.dtype_code(logits.dtype)
    device = logits.get_device()
    for x in (logits, tokens, *rows.values()):
        if x is not None and (x.get_device() != device or device < 0):
            if not (x.is_cuda and logits.is_cuda):
                raise RuntimeError("hip backend: tensors must live on the GPU (no CPU fallback)")
            raise ValueError(f"{what}: tensors on several devices")
    flat = {name: _row_values(x) for name, x in rows.items()}
    if len(shape) != 1:
        logits, tokens = logits.reshape(-1, logits.shape[-1]), tokens.reshape(-1)
    return logits, tokens if tokens.is_contiguous() else tokens.contiguous(), cap, flat


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_log_probs: torch.Tensor, advantages: torch.Tensor, *,
                ref_log_probs: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                clip: float | tuple[float, float] = 0.2, kl: float = 0.0,
                softcap: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, log_probs)``: the clipped policy loss (module docstring; a
    scalar, differentiable in the logits) and the tokens' present
    log-probabilities (fp32, without a gradient).

    ``logits`` [..., V] in bf16 or fp32, ``tokens`` int64 [...] (one outside [0, V)
    makes the loss NaN), ``old_log_probs`` and ``advantages`` [...], as
    ``ref_log_probs``, which the KL term needs (``kl`` > 0).  ``clip`` is the
    distance of the clipping borders from 1, below and above.  ``weights`` [...]
    multiplies each row's loss (default: the mean over all rows); a row of weight
    zero may hold anything in any input, and gives a log-probability of zero and a
    gradient of zero.  At most 2^24 rows (2^26 of up to 2048 logits) a call.
    ``softcap`` caps the logits at ``softcap tanh(z / softcap)``.  Forward-mode and
    second derivatives are refused.
    """
    low, high = (clip, clip) if isinstance(clip, (int, float)) else clip
    low, high, kl = float(low), float(high), float(kl)
    if not (0.0 <= low <= 1.0 and 0.0 <= high < float("inf")):
        raise ValueError(f"policy_loss: clip must lie in [0, 1] below and be at least 0 above, got {clip}")
    if not 0.0 <= kl < float("inf"):
        raise ValueError(f"policy_loss: kl must be at least 0, got {kl}")
    if kl and ref_log_probs is None:
        raise ValueError("policy_loss: the KL term needs ref_log_probs")
    if not torch.compiler.is_compiling():
        refuse_tangents("policy_loss", logits)
    z, tok, cap, r = _flat("policy_loss", logits, tokens, softcap,
                           {"old_log_probs": old_log_probs, "advantages": advantages,
                            "ref_log_probs": ref_log_probs if kl else None, "weights": weights})
    loss, lp, _ = _policy_op(z, tok, r["old_log_probs"], r["advantages"], r["ref_log_probs"], r["weights"], low, high,
                                kl, cap)
    lp = lp.detach()
    return loss, lp if tokens.ndim == 1 else lp.view(tokens.shape)


@torch.no_grad()
def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, *, softcap: float | None = None) -> torch.Tensor:
    """The tokens' log-probabilities [...] (fp32, without a gradient) under the
    (soft-capped) logits [..., V]: what :func:`policy_loss` takes as
    ``old_log_probs`` and ``ref_log_probs``, in the same arithmetic."""
    z, tok, cap, _ = _flat("token_log_probs", logits.detach(), tokens, softcap, {})
    if torch.compiler.is_compiling():  # (one opaque call, as the loss is)
        none = torch.zeros(z.shape[0], dtype=torch.float32, device=z.device)
        return _policy_op(z, tok, none, none, None, None, 0.0, 0.0, 0.0, cap)[1].view(tokens.shape)
    z = _rows(z)
    lp = torch.empty(z.shape[0], dtype=torch.float32, device=z.device)
    desc = _desc(z, cap)
    parts = torch.empty(_plan(z.shape[0], z.shape[1], desc.dtype, cap > 0.0)[0], dtype=torch.float64, device=z.device)
    io = _lib.PolicyIO(z.data_ptr(), tok.data_ptr(), None, None, None, None, lp.data_ptr(), None, None, parts.data_ptr(),
                       None, None)
    with _on(z.device), _lib.timed("ts_policy_loss_fwd", lambda: _lib.nbytes(z, tok, lp)):
        status = _lib.load().ts_policy_loss_fwd(ctypes.byref(desc), ctypes.byref(io), _lib.stream_handle(z.device))
    _lib.check(status, "ts_policy_loss_fwd")
    return lp.view(tokens.shape)
