"""Distillation from a teacher's top log-probabilities, on (soft-capped, tempered) logits.

Where :func:`.policy.policy_loss` learns from rollouts, this learns from a teacher that
names its K first tokens of each place with their log-probabilities: per row n, with
``x = cap tanh(z / cap) / temperature`` (or ``z / temperature``), ``lq = log softmax(x)``
and ``P_k = exp(lp_k)``::

    loss = sum_n w_n [ sum_k P_k (lp_k - lq_k) + P_r (log P_r - log Q_r) ]

``P_r = 1 - sum_k P_k`` and ``Q_r`` are the teacher's and the student's share of all other
tokens; without the tail, P is the softmax of the K log-probabilities (which may be any scores)
and the second term is left out; so it is where the student forbids all other tokens (logits of
-inf: what the teacher's log-probabilities leave there may be their rounding alone).  Where a
gradient is recorded, the forward's launch gives it too, for a unit upstream gradient
(ts_distill_fwd): it is as large as the logits and held to the backward, as a saved tensor, which
forms it again where the upstream gradient is another (as does a second backward of the same
loss).  A loss whose value alone is wanted is called without gradients.  No probabilities are
stored.  A row of weight zero is not read.
"""
from __future__ import annotations

import ctypes
import functools
import threading

import torch

from ... import _lib
from .delta import _on
from .dispatch import HipOp, eager_forward, refuse_tangents
from .policy import _capture, _row_values, _rows

MAX_LOGITS = 1 << 20


_GRADIENT = threading.local()  # the gradient that an eager forward leaves for its setup


@functools.lru_cache(maxsize=256)
def _plan(rows, stride, V, K, dtype, tail, cap, temperature, aligned) -> _lib.DistillDesc:
    return _lib.DistillDesc(rows, stride if rows > 1 else V, V, K, _lib.dtype_code(dtype), int(tail), cap, int(aligned),
                            temperature)


def _describe(z: torch.Tensor, K: int, tail: bool, cap: float, temperature: float) -> _lib.DistillDesc:
    rows, V = z.shape
    stride = z.stride(0)
    aligned = z.data_ptr() % 16 == 0 and (rows == 1 or stride * z.element_size() % 16 == 0)
    return _plan(rows, stride, V, K, z.dtype, tail, cap, temperature, aligned)


def _forward(z: torch.Tensor, ids: torch.Tensor, lps: torch.Tensor, weights: torch.Tensor | None, cap: float,
             temperature: float, tail: bool) -> list[torch.Tensor]:
    z = _rows(z)
    rows = z.shape[0]
    desc = _describe(z, ids.shape[1], tail, cap, temperature)
    loss = torch.empty((), dtype=torch.float32, device=z.device)
    each = torch.empty(rows, dtype=torch.float32, device=z.device)
    # parts of the loss (fp64), then what the backward takes of each row
    saved = torch.empty(7 * rows + 2, dtype=torch.float32, device=z.device)
    at = saved.data_ptr()
    dz = torch.empty(z.shape, dtype=z.dtype, device=z.device) if rows and eager_forward() else None
    io = _lib.DistillIO(z.data_ptr(), ids.data_ptr(), lps.data_ptr(), _lib.ptr(weights), each.data_ptr(), at + 8 * rows,
                        at, loss.data_ptr(), _lib.ptr(dz))
    with _on(z.device), _lib.timed("ts_distill_fwd", lambda: _lib.nbytes(z, ids, lps, weights, each, dz)):
        status = _lib.load().ts_distill_fwd(ctypes.byref(desc), ctypes.byref(io), _lib.stream_handle(z.device))
        graph = 0 if dz is None else _capture(z.device)
    _lib.check(status, "ts_distill_fwd")
    if dz is not None:
        _GRADIENT.of = (loss, dz, graph)
    return [loss, each, saved]


def _forward_fake(z, ids, lps, weights, cap, temperature, tail):
    return [z.new_empty((), dtype=torch.float32), z.new_empty(z.shape[0], dtype=torch.float32),
            z.new_empty(7 * z.shape[0] + 2, dtype=torch.float32)]


def _backward_impl(g: torch.Tensor, z: torch.Tensor, ids: torch.Tensor, lps: torch.Tensor,
                   weights: torch.Tensor | None, saved: torch.Tensor, cap: float, temperature: float,
                   tail: bool) -> torch.Tensor:
    return _gradient(g, z, ids, lps, weights, saved, cap, temperature, tail, None)


def _gradient(g, z, ids, lps, weights, saved, cap, temperature, tail, formed: torch.Tensor | None) -> torch.Tensor:
    """The logits' gradient; ``formed`` is the forward's, for a unit ``g``, which
    becomes it."""
    z = _rows(z)
    rows = z.shape[0]
    desc = _describe(z, ids.shape[1], tail, cap, temperature)
    dz = torch.empty(z.shape, dtype=z.dtype, device=z.device) if formed is None else formed
    g32 = g if g.dtype == torch.float32 else g.to(torch.float32)
    io = _lib.DistillIO(z.data_ptr(), ids.data_ptr(), lps.data_ptr(), _lib.ptr(weights), None,
                        saved.data_ptr() + 8 * rows, None, None, dz.data_ptr())
    lib, name = _lib.load(), "ts_distill_bwd" if formed is None else "ts_distill_scale"
    with _on(z.device), _lib.timed(name, lambda: _lib.nbytes(z, ids, lps, dz)):
        stream = _lib.stream_handle(z.device)
        if formed is None:
            status = lib.ts_distill_bwd(ctypes.byref(desc), ctypes.byref(io), g32.data_ptr(), dz.data_ptr(), stream)
        else:
            status = lib.ts_distill_scale(ctypes.byref(desc), ctypes.byref(io), g32.data_ptr(), stream)
    _lib.check(status, name)
    return dz


def _backward_fake(g, z, ids, lps, weights, saved, cap, temperature, tail):
    return z.new_empty(z.shape)


def _setup(ctx, inputs, output):
    z, ids, lps, weights, *ctx.settings = inputs
    left, _GRADIENT.of = getattr(_GRADIENT, "of", None), None
    dz, ctx.graph = left[1:] if left is not None and left[0] is output[0] else (None, None)
    ctx.save_for_backward(z, ids, lps, weights, output[2], dz)


def _backward(ctx, grads, bwd):
    if grads[0] is None:
        return (None,) * 7
    z, ids, lps, weights, saved, dz = ctx.saved_tensors
    graph, ctx.graph = ctx.graph, None
    if dz is not None and graph is not None:
        # (a backward in a graph of its own may be replayed more often than the
        # forward, and would take another gradient's for the unit one's; each is handed out once)
        with _on(dz.device):
            same = _capture(dz.device) == graph
        if same:
            # (.data: what the caller does with it is no change of the saved tensor)
            return (_gradient(grads[0], z, ids, lps, weights, saved, *ctx.settings, dz.data), *(None,) * 6)
    return (bwd(grads[0], z, ids, lps, weights, saved, *ctx.settings), *(None,) * 6)


_distill_op = HipOp("distill_loss", forward=_forward, forward_fake=_forward_fake, backward_impl=_backward_impl,
                    backward_fake=_backward_fake, setup=_setup, backward=_backward, once=True)


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, log_probs: torch.Tensor, *,
                 weights: torch.Tensor | None = None, temperature: float = 1.0, tail: bool = True,
                 softcap: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, each)``: the divergence of the student from its teacher (module docstring;
    a scalar, differentiable in the logits) and every row's own [...] before its weight
    (fp32, without a gradient).

    ``logits`` [..., V] in bf16 or fp32, V at most 2^20; ``ids`` int64 [..., K] the teacher's
    tokens in any order, ``log_probs`` [..., K] their log-probabilities (at the same
    temperature).  An id below zero is no token; one at or past V, or twice in a row, makes
    the row's loss and gradient NaN.  ``tail`` False leaves all other tokens out.
    A log-probability of -inf is a share of zero; without the tail, a row of none but those has no
    softmax and is NaN.  ``weights`` [...] multiplies each row's loss (default: the mean over all rows); a row of
    weight zero may hold anything in any input, and gives zero and a gradient of zero.
    ``softcap`` caps the logits at ``softcap tanh(z / softcap)``, before the temperature.
    At most 2^24 - 1 rows a call.  Forward-mode and second derivatives are refused.
    """
    what = "distill_loss"
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [..., V], got {tuple(logits.shape)}")
    V, shape = logits.shape[-1], tuple(logits.shape[:-1])
    if V > MAX_LOGITS:
        raise NotImplementedError(f"{what}: at most {MAX_LOGITS} logits a row, got {V}")
    if ids.ndim != logits.ndim or tuple(ids.shape[:-1]) != shape or ids.shape[-1] < 1 or ids.dtype != torch.int64:
        raise ValueError(f"{what}: ids must be int64 {shape + ('K',)}, got {ids.dtype} {tuple(ids.shape)}")
    if log_probs.shape != ids.shape or not log_probs.is_floating_point():
        raise ValueError(f"{what}: log_probs must be floating-point {tuple(ids.shape)}, got {log_probs.dtype} "
                         f"{tuple(log_probs.shape)}")
    if weights is not None and tuple(weights.shape) != shape:
        raise ValueError(f"{what}: weights must be {shape}, got {tuple(weights.shape)}")
    cap = 0.0 if softcap is None else float(softcap)
    if softcap is not None and not 1e-29 <= cap <= 1e29:
        raise ValueError(f"{what}: softcap must be positive, in [1e-29, 1e29] (None: no cap), got {softcap}")
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{what}: temperature must lie in [1e-6, 1e6], got {temperature}")
    _lib.dtype_code(logits.dtype)
    if not torch.compiler.is_compiling():
        refuse_tangents(what, logits)
    device = logits.get_device()
    for x in (logits, ids, log_probs, weights):
        if x is not None and (x.get_device() != device or device < 0):
            if not (x.is_cuda and logits.is_cuda):
                raise RuntimeError("hip backend: tensors must live on the GPU (no CPU fallback)")
            raise ValueError(f"{what}: tensors on several devices")
    z, ids = logits.reshape(-1, V), ids.reshape(-1, ids.shape[-1]).contiguous()
    lps = log_probs.detach().to(torch.float32).reshape(ids.shape).contiguous()
    loss, each, _ = _distill_op(z, ids, lps, _row_values(weights), cap, temperature, bool(tail))
    return loss, each.detach().view(shape)
