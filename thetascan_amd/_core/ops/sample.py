"""Sampling of tokens from (soft-capped) logits, from given random numbers.

What a rollout draws its tokens with, and what :func:`.policy.policy_loss` then takes of
them: per row of the logits, with ``y = cap tanh(z / cap)`` (or z)::

    w_i = round(2^44 exp((y_i - max y) / temperature))

Left are the ``top_k`` highest logits (ties: the lowest index first); of those, in that
order, the tokens with less than ``top_p`` of their weight before them; of those, the ones
of at least ``min_p`` of the highest token's weight.  The token is the first, by index,
whose running weight is over ``floor(u total)``.  The weights are whole numbers, so that
the token is the same however the sums are split.  One launch (ts_sample_tokens), a
workgroup a row.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ... import _lib
from .delta import _on
from .dispatch import refuse_tangents
from .policy import _rows

MAX_TOKENS = (1 << 19) - 1  # (their weights add up in 63 bits)


def _setting(name: str, x, rows: tuple, least: float, none: float, whole: bool = False):
    """A setting as (one for all rows, or a tensor of one a row)."""
    what = "sample_tokens"
    if isinstance(x, torch.Tensor):
        if tuple(x.shape) != rows or x.dtype == torch.bool or x.is_floating_point() == whole or x.is_complex():
            raise ValueError(f"{what}: {name} must be {'integers' if whole else 'floating-point'} {rows}, "
                             f"got {x.dtype} {tuple(x.shape)}")
        return none, x.detach().to(torch.int64 if whole else torch.float32).reshape(-1).contiguous()
    if x is None:
        return none, None
    if isinstance(x, bool) or not isinstance(x, int if whole else (int, float)) or not x >= least or math.isinf(x):
        raise ValueError(f"{what}: {name} must be {'a whole number' if whole else 'a number'} of at least {least}, "
                         f"got {x!r}")
    return x, None


@torch.no_grad()
def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor | None = None, top_p: float | torch.Tensor | None = None,
                  min_p: float | torch.Tensor | None = None,
                  softcap: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(tokens, log_probs)``: a token of each row (int64; module docstring) and its
    log-probability under all of the (soft-capped) logits at temperature one (fp32), which
    is what :func:`.policy.policy_loss` takes as ``old_log_probs``.

    ``logits`` [..., V] in bf16 or fp32, V below 2^19; ``uniforms`` [...] random numbers
    in [0, 1).  ``temperature`` (0: the highest logit), ``top_k``, ``top_p`` and ``min_p``
    are one for all rows or tensors [...] (fp32, ``top_k`` of integers); None: no cut.  In
    tensors, a ``top_k`` below one counts as one, a ``top_p`` at or below zero leaves the
    first token, a ``min_p`` over one counts as one.  ``softcap`` caps the logits at
    ``softcap tanh(z / softcap)``.  A logit of -inf is no token, whatever the cap; a row that has no
    token, or +inf or NaN in it, or a temperature below zero, or a setting that is NaN, gives
    token -1 and NaN.  Fewer than 2^22 rows a call.
    """
    what = "sample_tokens"
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [..., V], got {tuple(logits.shape)}")
    V, shape = logits.shape[-1], tuple(logits.shape[:-1])
    if V > MAX_TOKENS:
        raise NotImplementedError(f"{what}: at most {MAX_TOKENS} tokens, got {V}")
    if tuple(uniforms.shape) != shape or not uniforms.is_floating_point():
        raise ValueError(f"{what}: uniforms must be floating-point {shape}, got {uniforms.dtype} {tuple(uniforms.shape)}")
    cap = 0.0 if softcap is None else float(softcap)
    if softcap is not None and not 1e-29 <= cap <= 1e29:
        raise ValueError(f"{what}: softcap must be positive, in [1e-29, 1e29] (None: no cap), got {softcap}")
    code = _lib.dtype_code(logits.dtype)
    if torch.compiler.is_compiling():
        raise NotImplementedError(f"{what}: not under torch.compile")
    refuse_tangents(what, logits)
    t, ts = _setting("temperature", temperature, shape, 0, 1.0)
    k, ks = _setting("top_k", top_k, shape, 1, V, True)
    p, ps = _setting("top_p", top_p, shape, 0, 1.0)
    m, ms = _setting("min_p", min_p, shape, 0, 0.0)
    device = logits.get_device()
    for x in (logits, uniforms, ts, ks, ps, ms):
        if x is not None and (x.get_device() != device or device < 0):
            if not (x.is_cuda and logits.is_cuda):
                raise RuntimeError("hip backend: tensors must live on the GPU (no CPU fallback)")
            raise ValueError(f"{what}: tensors on several devices")
    z = _rows(logits.detach().reshape(-1, V))
    u = uniforms.detach().to(torch.float32).reshape(-1).contiguous()
    rows = z.shape[0]
    tokens = torch.empty(rows, dtype=torch.int64, device=z.device)
    log_probs = torch.empty(rows, dtype=torch.float32, device=z.device)
    desc = _lib.SampleDesc(rows, z.stride(0) if rows > 1 else V, V, code, cap, 0, t, p, m, min(k, V))
    io = _lib.SampleIO(z.data_ptr(), u.data_ptr(), _lib.ptr(ts), _lib.ptr(ps), _lib.ptr(ms), _lib.ptr(ks),
                       tokens.data_ptr(), log_probs.data_ptr())
    with _on(z.device), _lib.timed("ts_sample_tokens", lambda: _lib.nbytes(z, u, tokens, log_probs)):
        status = _lib.load().ts_sample_tokens(ctypes.byref(desc), ctypes.byref(io), _lib.stream_handle(z.device))
    _lib.check(status, "ts_sample_tokens")
    return tokens.view(shape), log_probs.view(shape)
