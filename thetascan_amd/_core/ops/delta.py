"""The gated delta rule: a causal memory that writes what it does not yet know.

:func:`gated_delta_rule` is the error-correcting counterpart of the additive
scans (:func:`.scan_hip.linattn`), with the same streams and retentions.  From
the fp32 state ``S`` [dk, dv] of a value head, token after token::

    S <- a_t S                        # the retention, a = exp(log a)
    u  = beta_t (v_t - S^T k_t)       # what the memory misses, times the write strength
    S <- S + k_t u^T
    out_t = S^T q_t

Whole sequences run in chunks of 64 tokens on MFMA (ts_delta_fwd, with
ts_delta_bwd for the gradients); a few tokens against a carried state, without
gradients, run token by token in one pass over the state (ts_delta_step).  Both
are the same function of their inputs.

bf16 inputs: products take bf16 operands and fp32 sums; what is not an input enters in
three bf16 parts in the forward, so the returned state is one of fp32 arithmetic, and in
two in the backward: bf16 outputs and gradients carry bf16's one rounding, fp32 gradients
(of states and of fp32 gates) 16 bits.  fp32 inputs compute in fp32.
A value that is not finite reaches no output before its own token; from there on outputs
and the state are not finite (of its value column where it stands in v, of its own token
where in q).  Gradients of its chunk of 64 tokens and of the tokens before are not either.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import torch

from ... import _lib
from .dispatch import HipOp, refuse_tangents
from .scan_hip import _kernel_view, _vec

MAX_KEYS, MAX_VALUES = 128, 512
# Tokens that the recurrent form takes (without gradients).  Its time grows with the
# tokens, the chunked form's does not (to 64): 16 heads of 64 x 64 4.3 us for one token, 11.6
# for 12, 14.2 for 16 against 15.4; 128 of 128 x 128 7, 18.9 and 23.0 against 22; 2048 of
# those 49, 96 and 117 against 154.
STEP_TOKENS = 12


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """The device a launch needs as the current one (a no-op where it is)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(device)


def _width(dtype: torch.dtype, n: int) -> int:
    vec = _vec(dtype)
    return -(-n // vec) * vec


def _gate(t: torch.Tensor | None, heads: bool = False) -> _lib.Strided:
    if t is None:
        return _lib.Strided(None, 0, 0, 0)
    if heads:
        return _lib.Strided(t.data_ptr(), 0, t.stride(0), 0)
    return _lib.Strided(t.data_ptr(), *t.stride())


def _describe(q, v, dtype, beta, decay, keep) -> _lib.DeltaDesc:
    B, Hk, T, dk = q
    return _lib.DeltaDesc(B, Hk, v[1], T, _width(dtype, dk), _width(dtype, v[3]), _lib.dtype_code(dtype),
                          _lib.dtype_code(beta), _lib.TS_F32 if decay is None else _lib.dtype_code(decay), int(keep))


def _desc(q, k, v, beta, decay, keep: bool) -> _lib.DeltaDesc:
    """The descriptor of a call with these tensors, the caller's own."""
    return _describe(q.shape, v.shape, q.dtype, beta.dtype, None if decay is None else decay.dtype, keep)


@functools.lru_cache(maxsize=256)
def _plan(q, v, dtype, beta, decay, keep) -> tuple[_lib.DeltaDesc, int, int, int]:
    """A call's descriptor and the bytes of its forward's workspace, of the low
    halves beside it and of the backward's workspace, by shapes and dtypes."""
    desc = _describe(q, v, dtype, beta, decay, keep)
    lib, fwd, low, bwd = _lib.load(), ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    _lib.check(lib.ts_delta_workspace_bytes(ctypes.byref(desc), ctypes.byref(fwd)), "ts_delta_workspace_bytes")
    _lib.check(lib.ts_delta_low_bytes(ctypes.byref(desc), ctypes.byref(low)), "ts_delta_low_bytes")
    _lib.check(lib.ts_delta_bwd_workspace_bytes(ctypes.byref(desc), ctypes.byref(bwd)), "ts_delta_bwd_workspace_bytes")
    return desc, fwd.value, low.value, bwd.value


def _rows(x: torch.Tensor, vec: int) -> tuple[torch.Tensor, _lib.Strided]:
    """``x`` (or its copy) as the kernels read it, and its description."""
    s = x.stride()
    if s[3] != 1 or (s[0] | s[1] | s[2]) % vec or x.shape[3] % vec or x.data_ptr() % 16:
        x = _kernel_view(x)
        s = x.stride()
    return x, _lib.Strided(x.data_ptr(), s[0], s[1], s[2])


def _padded_state(state: torch.Tensor | None, dk: int, dv: int) -> torch.Tensor | None:
    if state is None:
        return None
    if state.shape[-2:] == (dk, dv) and state.is_contiguous() and state.data_ptr() % 16 == 0:
        return state
    out = state.new_zeros(*state.shape[:2], dk, dv)
    out[..., :state.shape[-2], :state.shape[-1]] = state
    return out


def _rows_like(x: torch.Tensor, dtype: torch.dtype, width: int) -> torch.Tensor:
    """[B,H,T,width] in x's own order: token-major memory for a projection's heads."""
    B, H, T, _ = x.shape
    if H > 1 and T > 1 and x.stride(1) < x.stride(2):
        return x.new_empty(B, T, H, width, dtype=dtype).transpose(1, 2)
    return x.new_empty(B, H, T, width, dtype=dtype)


def _io(q, k, v, beta, decay, lengths, out, state, state_out, low=None) -> _lib.DeltaIO:
    """(q, k, v and out by their descriptions)"""
    return _lib.DeltaIO(q, k, v, _gate(beta), _gate(decay, decay is not None and decay.ndim == 1), out,
                        _lib.ptr(lengths), _lib.ptr(state), _lib.ptr(state_out), low)


def _launch(q, k, v, beta, decay, state, lengths, want_state: bool, keep: bool, step: bool, state_out=None):
    """``(out, state or None, workspace or None)`` at the padded widths' slices."""
    lib = _lib.load()
    desc, nbytes, low, _ = _plan(q.shape, v.shape, q.dtype, beta.dtype, None if decay is None else decay.dtype, keep)
    B, H, T, dv = v.shape
    dk, dkp, dvp, vec = q.shape[-1], desc.dk, desc.dv, _vec(q.dtype)
    (q, sq), (k, sk), (v4, sv) = _rows(q, vec), _rows(k, vec), _rows(v, vec)
    out = _rows_like(v, q.dtype, dvp)
    given = _padded_state(state, dkp, dvp)
    final = None
    if want_state:
        if state_out is not None and (dkp, dvp) == (dk, dv) and state_out.data_ptr() % 16 == 0:
            final = state_out
        else:
            final = torch.empty(B, H, dkp, dvp, dtype=torch.float32, device=q.device)
    io = _io(sq, sk, sv, beta, decay, lengths, _lib.strided(out), given, final)
    work = None
    with _on(q.device):
        stream = _lib.stream_handle(q.device)
        if step:
            with _lib.timed("ts_delta_step", lambda: _lib.nbytes(q, k, v4, out, given, final)):
                status = lib.ts_delta_step(ctypes.byref(desc), ctypes.byref(io), stream)
            _lib.check(status, "ts_delta_step")
        else:
            work = torch.empty(nbytes + low, dtype=torch.uint8, device=q.device)
            io.low = work.data_ptr() + nbytes if low else None
            with _lib.timed("ts_delta_fwd", lambda: _lib.nbytes(q, k, v4, beta, decay, out, given, final)):
                status = lib.ts_delta_fwd(ctypes.byref(desc), ctypes.byref(io), work.data_ptr(), nbytes, stream)
            _lib.check(status, "ts_delta_fwd")
    if final is not None and final is state_out and not final.is_inference():
        # (the kernel's writing is autograd's in-place change: what saved the old values says so)
        torch.autograd.graph.increment_version(final)
    if final is not None and final is not state_out:
        final = final[..., :dk, :dv]
        if (dkp, dvp) != (dk, dv):
            final = final.contiguous()
        if state_out is not None:
            final = state_out.copy_(final)
    return out if dvp == dv else out[..., :dv], final, work


def _forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: torch.Tensor, decay: torch.Tensor | None,
             state: torch.Tensor | None, lengths: torch.Tensor | None, want_state: bool, keep: bool,
             step: bool) -> list[torch.Tensor]:
    out, final, work = _launch(q, k, v, beta, decay, state, lengths, want_state, keep, step)
    none = q.new_empty(0, dtype=torch.float32)
    return [out, none if final is None else final, work if keep else q.new_empty(0, dtype=torch.uint8)]


def _forward_fake(q, k, v, beta, decay, state, lengths, want_state, keep, step):
    B, H, _, dv = v.shape
    out = _rows_like(v, q.dtype, _width(q.dtype, dv))[..., :dv]
    nbytes = 0
    if keep:  # (a traced size becomes a number here)
        nbytes = sum(_plan(tuple(map(int, q.shape)), tuple(map(int, v.shape)), q.dtype, beta.dtype,
                           None if decay is None else decay.dtype, True)[1:3])
    return [out, q.new_empty((B, H, q.shape[-1], dv) if want_state else (0,), dtype=torch.float32),
            q.new_empty(nbytes, dtype=torch.uint8)]


def _backward_impl(dout: torch.Tensor | None, dfinal: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor,
                   v: torch.Tensor, beta: torch.Tensor, decay: torch.Tensor | None, state: torch.Tensor | None,
                   lengths: torch.Tensor | None, saved: torch.Tensor, need_state: bool) -> list[torch.Tensor]:
    lib = _lib.load()
    desc, kept, low, nbytes = _plan(q.shape, v.shape, q.dtype, beta.dtype, None if decay is None else decay.dtype, True)
    B, H, T, dv = v.shape
    dk, dkp, dvp, vec = q.shape[-1], desc.dk, desc.dv, _vec(q.dtype)
    (q4, sq), (k4, sk), (v4, sv) = _rows(q, vec), _rows(k, vec), _rows(v, vec)
    if dout is None:
        dout = torch.zeros(B, H, T, dvp, dtype=q.dtype, device=q.device)
    do4, so = _rows(dout if dout.dtype == q.dtype else dout.to(q.dtype), vec)
    given = None if dfinal is None else _padded_state(dfinal.to(torch.float32), dkp, dvp)
    dq, dk_, dv_ = _rows_like(q, q.dtype, dkp), _rows_like(k, q.dtype, dkp), _rows_like(v, q.dtype, dvp)
    dbeta = torch.empty(B, H, T, dtype=beta.dtype, device=q.device)
    per_head = decay is not None and decay.ndim == 1
    ddecay = None
    if decay is not None:
        ddecay = torch.empty((H,) if per_head else (B, H, T), dtype=decay.dtype, device=q.device)
    dstate = torch.empty(B, H, dkp, dvp, dtype=torch.float32, device=q.device) if need_state else None
    # (the forward's output and states play no part here: out takes dout's rows)
    io = _io(sq, sk, sv, beta, decay, lengths, so, None, None, saved.data_ptr() + kept if low else None)
    grads = _lib.DeltaGrads(so, _lib.strided(dq), _lib.strided(dk_), _lib.strided(dv_), dbeta.data_ptr(),
                            None if per_head else _lib.ptr(ddecay), _lib.ptr(ddecay) if per_head else None,
                            _lib.ptr(given), _lib.ptr(dstate))
    work = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    with _on(q.device), _lib.timed("ts_delta_bwd", lambda: _lib.nbytes(q4, k4, v4, do4, dq, dk_, dv_, dbeta, ddecay)):
        status = lib.ts_delta_bwd(ctypes.byref(desc), ctypes.byref(io), ctypes.byref(grads), saved.data_ptr(),
                                  kept, work.data_ptr(), work.numel(), _lib.stream_handle(q.device))
    _lib.check(status, "ts_delta_bwd")
    if (dkp, dvp) != (dk, dv):
        dq, dk_, dv_ = dq[..., :dk], dk_[..., :dk], dv_[..., :dv]
        dstate = None if dstate is None else dstate[..., :dk, :dv].contiguous()
    return [dq, dk_, dv_, dbeta, q.new_empty(0) if ddecay is None else ddecay,
            q.new_empty(0, dtype=torch.float32) if dstate is None else dstate]


def _backward_fake(dout, dfinal, q, k, v, beta, decay, state, lengths, saved, need_state):
    def rows(x):
        return _rows_like(x, q.dtype, _width(q.dtype, x.shape[-1]))[..., :x.shape[-1]]

    B, H, _, dv = v.shape
    return [rows(q), rows(k), rows(v), beta.new_empty(beta.shape),
            q.new_empty(0) if decay is None else decay.new_empty(decay.shape),
            q.new_empty((B, H, q.shape[-1], dv) if need_state else (0,), dtype=torch.float32)]


def _setup(ctx, inputs, output):
    q, k, v, beta, decay, state, lengths, want_state, keep, step = inputs
    ctx.need_state = state is not None and state.requires_grad
    ctx.want_state = want_state
    ctx.need_decay = decay is not None and decay.requires_grad
    ctx.save_for_backward(q, k, v, beta, decay, state, lengths, output[2])


def _backward(ctx, grads, bwd):
    q, k, v, beta, decay, state, lengths, saved = ctx.saved_tensors
    dout, dfinal = grads[0], grads[1] if ctx.want_state else None
    if dout is None and dfinal is None:
        return (None,) * 10
    dq, dk, dv, dbeta, ddecay, dstate = bwd(dout, dfinal, q, k, v, beta, decay, state, lengths, saved, ctx.need_state)
    return (dq, dk, dv, dbeta, ddecay if ctx.need_decay else None, dstate if ctx.need_state else None, None, None, None,
            None)


_delta_op = HipOp("gated_delta", forward=_forward, forward_fake=_forward_fake, backward_impl=_backward_impl,
                  backward_fake=_backward_fake, setup=_setup, backward=_backward, once=True)


def _token_gate(t: torch.Tensor, name: str, B: int, H: int, T: int) -> torch.Tensor:
    if t.ndim == 4 and t.shape[-1] == 1:
        t = t.squeeze(-1)
    if tuple(t.shape) != (B, H, T):
        raise ValueError(f"gated_delta_rule: {name} must be [B,H,T] or [B,H,T,1] = {(B, H, T)}, got {tuple(t.shape)}")
    return t


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: torch.Tensor,
                     retention: torch.Tensor | None = None, *, state: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None, return_state: bool = False,
                     state_out: torch.Tensor | None = None):
    """Outputs [B,H,T,dv] of the gated delta rule (module docstring), and with
    ``return_state`` the fp32 state [B,H,dk,dv] after the last token.

    ``q``, ``k`` [B,Hk,T,dk] and ``v`` [B,H,T,dv] (bf16 or fp32, any strides; H a
    multiple of Hk: value head h reads the keys and queries of head h // (H / Hk));
    ``beta`` [B,H,T] or [B,H,T,1] the write strengths; ``retention`` the log
    retentions (at most zero, -inf a reset): None, one per value head [H], or one
    per token [B,H,T] or [B,H,T,1].  Keys are taken as given: the memory is stable
    where ``beta_t |k_t|^2`` is at most 2, and keeps its digits to there (with alike
    keys and no retention, bf16 gradients are off by 3e-5 of their norm before their
    rounding at 0.5 to 2, fp32's by 2e-5 at 2).  dk is at
    most 128, dv at most 512.

    ``state`` continues from the fp32 state of an earlier call (None: zero).
    ``lengths`` [B] (integers, on the GPU, clamped to [0, T]) makes a padded batch:
    tokens at or past a sequence's length are not read, give zeros and gradients of
    zero, and leave its state as it was.  ``state_out`` (without gradients only) is
    the contiguous fp32 tensor to write the new state into; it may be ``state``.

    Differentiable in q, k, v, beta, the retention and the state (once, backwards:
    forward-mode and second derivatives are refused).
    """
    if not q.ndim == k.ndim == v.ndim == 4:
        name, x = next(i for i in (("q", q), ("k", k), ("v", v)) if i[1].ndim != 4)
        raise ValueError(f"gated_delta_rule: {name} must be [B,H,T,D], got {tuple(x.shape)}")
    (B, Hk, T, dk), (Bv, H, Tv, dv) = q.shape, v.shape
    if k.shape != q.shape or Bv != B or Tv != T:
        raise ValueError(f"gated_delta_rule: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if min(B, Hk, dk, dv, H) < 1 or H % Hk:
        raise ValueError(f"gated_delta_rule: {H} value heads over {Hk} key heads, {B} sequences, widths {dk} and {dv}")
    if dk > MAX_KEYS or dv > MAX_VALUES:
        raise NotImplementedError(f"gated_delta_rule: at most {MAX_KEYS} keys and {MAX_VALUES} values, got {dk} and {dv}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"gated_delta_rule: q, k and v of one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    beta = _token_gate(beta, "beta", B, H, T)
    if retention is not None and retention.ndim == 1:
        if retention.numel() != H:
            raise ValueError(f"gated_delta_rule: a static retention has one entry per value head ({H}), "
                             f"got {retention.numel()}")
    elif retention is not None:
        if retention.ndim == 4 and retention.shape[-1] != 1:
            raise NotImplementedError("gated_delta_rule: one retention per token and head (no per-channel decay)")
        retention = _token_gate(retention, "retention", B, H, T)
    for x in (q, beta, retention):
        if x is not None:
            _lib.dtype_code(x.dtype)
    for name, s in (("state", state), ("state_out", state_out)):
        if s is not None and (tuple(s.shape) != (B, H, dk, dv) or s.dtype != torch.float32):
            raise ValueError(f"gated_delta_rule: {name} must be fp32 {(B, H, dk, dv)}, got {s.dtype} {tuple(s.shape)}")
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"gated_delta_rule: lengths must be integers [{B}], got {lengths.dtype} {tuple(lengths.shape)}")
    if not torch.compiler.is_compiling():
        refuse_tangents("gated_delta_rule", q, k, v, beta, retention, state)
    device, record = q.get_device(), torch.is_grad_enabled() and q.requires_grad
    if device < 0:
        raise RuntimeError("hip backend: tensors must live on the GPU (no CPU fallback)")
    for x in (k, v, beta, retention, state, lengths, state_out):
        if x is not None:
            if x.get_device() != device:
                if not x.is_cuda:
                    raise RuntimeError("hip backend: tensors must live on the GPU (no CPU fallback)")
                raise ValueError("gated_delta_rule: tensors on several devices")
            record = record or (x.requires_grad and torch.is_grad_enabled())
    if lengths is not None:
        lengths = lengths.to(torch.int64).contiguous()
    if state_out is not None:
        if record or state_out.requires_grad:
            raise ValueError("gated_delta_rule: state_out takes no part in gradients: call it without them")
        if not state_out.is_contiguous():
            raise ValueError("gated_delta_rule: state_out must be contiguous")
        # (a head's new state would meet another's old one; a state that is not contiguous is read from a copy)
        if state is not None and state.is_contiguous() and (
                0 < abs(state_out.data_ptr() - state.data_ptr()) < 4 * state.numel()):
            raise ValueError("gated_delta_rule: state_out overlaps the state (it may be the state itself)")
        if torch.compiler.is_compiling():
            raise NotImplementedError("gated_delta_rule: a traced call writes into no tensor it is given (state_out)")
    if T == 0:
        final = torch.zeros(B, H, dk, dv, dtype=torch.float32, device=q.device) if state is None else state.clone()
        if state_out is not None:
            final = state_out.copy_(final)
        out = v.new_empty(B, H, 0, dv)
        return (out, final) if return_state else out
    step = not record and T <= STEP_TOKENS
    if state_out is not None or not (record or torch.compiler.is_compiling()):
        out, final, _ = _launch(q, k, v, beta, retention, state, lengths, return_state or state_out is not None, False,
                                step, state_out)
        return (out, final) if return_state else out
    out, final, _ = _delta_op(q, k, v, beta, retention, state, lengths, bool(return_state), record, step)
    return (out, final) if return_state else out
