"""Distillation from a teacher's top log-probabilities, on (soft-capped, tempered) logits.

Where :func:`.policy.policy_loss` learns from rollouts, this learns from a teacher that
names its K first tokens of each place with their log-probabilities: per row n, with
``x = cap tanh(z / cap) / temperature`` (or ``z / temperature``), ``lq = log softmax(x)``
and ``P_k = exp(lp_k)``::

    loss = sum_n w_n [ sum_k P_k (lp_k - lq_k) + P_r (log P_r - log Q_r) ]

``P_r = 1 - sum_k P_k`` and ``Q_r`` are the teacher's and the student's share of all other
tokens; without the tail, P is the softmax of the K log-probabilities and the second term
is left out.  One pass over the logits a direction (ts_distill_fwd, ts_distill_bwd); no
probabilities are stored.  A row of weight zero is not read.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from ... import _lib
from .delta import _on
from .dispatch import HipOp, refuse_tangents
from .policy import _row_values, _rows

MAX_LOGITS = 1 << 20


@functools.lru_cache(maxsize=256)
def _describe(rows, stride, V, K, dtype, tail, cap, temperature) -> tuple[_lib.DistillDesc, int]:
    """A call's description and the partial sums of its loss."""
    desc = _lib.DistillDesc(rows, stride if rows > 1 else V, V, K, _lib.dtype_code(dtype), int(tail), cap, 0, temperature)
    n = ctypes.c_int64()
    _lib.check(_lib.load().ts_distill_parts(ctypes.byref(desc), ctypes.byref(n)), "ts_distill_parts")
    return desc, n.value


def _forward(z: torch.Tensor, ids: torch.Tensor, lps: torch.Tensor, weights: torch.Tensor | None, cap: float,
             temperature: float, tail: bool) -> list[torch.Tensor]:
    z = _rows(z)
    rows, V = z.shape
    desc, parts = _describe(rows, z.stride(0), V, ids.shape[1], z.dtype, tail, cap, temperature)
    loss = torch.empty((), dtype=torch.float32, device=z.device)
    each = torch.empty(rows, dtype=torch.float32, device=z.device)
    # the parts of the loss (fp64), then what the backward takes of each row
    saved = torch.empty(max(2 * parts + 4 * rows, 2), dtype=torch.float32, device=z.device)
    at = saved.data_ptr()
    io = _lib.DistillIO(z.data_ptr(), ids.data_ptr(), lps.data_ptr(), _lib.ptr(weights), each.data_ptr(), at + 8 * parts,
                        at, loss.data_ptr())
    with _on(z.device), _lib.timed("ts_distill_fwd", lambda: _lib.nbytes(z, ids, lps, weights, each)):
        status = _lib.load().ts_distill_fwd(ctypes.byref(desc), ctypes.byref(io), _lib.stream_handle(z.device))
    _lib.check(status, "ts_distill_fwd")
    return [loss, each, saved]


def _forward_fake(z, ids, lps, weights, cap, temperature, tail):
    # (a traced size becomes a number here: the parts follow no formula of it)
    parts = _describe(int(z.shape[0]), int(z.shape[1]), int(z.shape[1]), int(ids.shape[1]), z.dtype, tail, cap,
                      temperature)[1]
    return [z.new_empty((), dtype=torch.float32), z.new_empty(z.shape[0], dtype=torch.float32),
            z.new_empty(max(2 * parts + 4 * z.shape[0], 2), dtype=torch.float32)]


def _backward_impl(g: torch.Tensor, z: torch.Tensor, ids: torch.Tensor, lps: torch.Tensor,
                   weights: torch.Tensor | None, saved: torch.Tensor, cap: float, temperature: float,
                   tail: bool) -> torch.Tensor:
    z = _rows(z)
    rows, V = z.shape
    desc, _ = _describe(rows, z.stride(0), V, ids.shape[1], z.dtype, tail, cap, temperature)
    dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    g32 = g if g.dtype == torch.float32 else g.to(torch.float32)
    io = _lib.DistillIO(z.data_ptr(), ids.data_ptr(), lps.data_ptr(), _lib.ptr(weights), None,
                        saved.data_ptr() + 4 * (saved.numel() - 4 * rows), None, None)
    with _on(z.device), _lib.timed("ts_distill_bwd", lambda: _lib.nbytes(z, ids, lps, dz)):
        status = _lib.load().ts_distill_bwd(ctypes.byref(desc), ctypes.byref(io), g32.data_ptr(), dz.data_ptr(),
                                            _lib.stream_handle(z.device))
    _lib.check(status, "ts_distill_bwd")
    return dz


def _backward_fake(g, z, ids, lps, weights, saved, cap, temperature, tail):
    return z.new_empty(z.shape)


def _setup(ctx, inputs, output):
    z, ids, lps, weights, *ctx.settings = inputs
    ctx.save_for_backward(z, ids, lps, weights, output[2])


def _backward(ctx, grads, bwd):
    if grads[0] is None:
        return (None,) * 7
    z, ids, lps, weights, saved = ctx.saved_tensors
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
    ``weights`` [...] multiplies each row's loss (default: the mean over all rows); a row of
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
