"""A token mixer whose memory learns by the gated delta rule.

:class:`GatedDelta` has the ``[batch, time, channels]`` contract of
:class:`thetascan_amd.ThetaScan` and a state of the same kind: whole sequences
(with gradients), continuation from a state, and one-token steps that
:class:`thetascan_amd.DecodeGraph` captures.
"""
from __future__ import annotations

import dataclasses

import torch
import torch.nn as nn
import torch.nn.functional as F

from ._core.modules.gates import DecayGate, OutGate, _HeadLinear
from ._core.ops import prologue, rownorm, stream
from ._core.ops.delta import MAX_KEYS, gated_delta_rule
from ._core.ops.linear import keeps_dtype, linear
from .state import ThetaScanState, config_fingerprint

_EPS = 1e-6


@dataclasses.dataclass(frozen=True)
class GatedDeltaConfig:
    """``n_heads`` value heads of ``d_model / n_heads`` channels; ``key_heads``
    key and query heads (None: one per value head) of the same width, each shared
    by ``n_heads / key_heads`` value heads."""

    d_model: int
    n_heads: int
    key_heads: int | None = None

    @property
    def head_dim(self) -> int:
        return self.d_model // self.n_heads

    def validate(self) -> None:
        if self.d_model < 1 or self.n_heads < 1 or self.d_model % self.n_heads:
            raise ValueError(f"d_model ({self.d_model}) must be a multiple of n_heads ({self.n_heads})")
        if self.key_heads is not None and (self.key_heads < 1 or self.n_heads % self.key_heads):
            raise ValueError(f"n_heads ({self.n_heads}) must be a multiple of key_heads ({self.key_heads})")
        if self.head_dim > MAX_KEYS:
            raise NotImplementedError(f"heads of at most {MAX_KEYS} channels, got {self.head_dim}")


def _l2norm(x: torch.Tensor) -> torch.Tensor:
    y = prologue.qk_norm(x, 0, 1.0, _EPS)
    return F.normalize(x.float(), dim=-1, eps=_EPS).to(x.dtype) if y is None else y


def _linear(x: torch.Tensor, lin: nn.Linear) -> torch.Tensor:
    # (the split-K gradients take one dtype throughout: under an autocast to
    # another the products and their gradients are torch's)
    if keeps_dtype(x.dtype) and lin.weight.dtype == x.dtype:
        return linear(x, lin.weight, lin.bias)
    return F.linear(x, lin.weight, lin.bias)


class GatedDelta(nn.Module):
    """``proj_out(silu(gate(x)) * rms_norm(memory))`` with the memory's outputs
    :func:`thetascan_amd.gated_delta_rule` of L2-normalized queries and keys, a
    write strength ``sigmoid(W x + b)`` and a retention ``exp(-softplus(W x + b))``
    per token and head."""

    def __init__(self, config: GatedDeltaConfig):
        super().__init__()
        config.validate()
        self.cfg = config
        keys = (config.key_heads or config.n_heads) * config.head_dim
        self.proj_q = nn.Linear(config.d_model, keys, bias=False)
        self.proj_k = nn.Linear(config.d_model, keys, bias=False)
        self.proj_v = nn.Linear(config.d_model, config.d_model, bias=False)
        self.beta = _HeadLinear(config.d_model, config.n_heads, 1, bias_init=0.0)
        self.decay = DecayGate(config.d_model, config.n_heads)
        self.ogate = OutGate(config.d_model, config.n_heads, config.head_dim)
        self.proj_out = nn.Linear(config.d_model, config.d_model, bias=False)

    def initial_state(self) -> ThetaScanState:
        """The state of a sequence with no tokens yet."""
        return ThetaScanState(fingerprint=config_fingerprint(self.cfg))

    def forward(self, x: torch.Tensor, state: ThetaScanState | None = None, *, lengths: torch.Tensor | None = None):
        """``y`` [B,T,D]; with ``state`` the sequence continues from it (without
        autograd) and ``(y, new_state)`` is returned.  ``lengths`` [B] makes a
        padded batch: tokens at or past a sequence's length are not read (whatever they
        hold), write nothing, and their outputs are zero."""
        if state is None:
            if lengths is not None:
                if tuple(lengths.shape) != x.shape[:1]:
                    raise ValueError(f"lengths must be [{x.shape[0]}], got {tuple(lengths.shape)}")
                # (what the padding holds must not meet the projections, nor their gradients)
                past = torch.arange(x.shape[1], device=x.device) >= lengths.unsqueeze(1)
                x = x.masked_fill(past.unsqueeze(-1), 0.0)
            return self._mix(x, None, None, lengths)[0] if x.shape[1] else torch.zeros_like(x)
        if lengths is not None:
            raise ValueError("a state counts one position for every sequence: a continued call takes no lengths")
        if state.fingerprint != config_fingerprint(self.cfg):
            raise ValueError("this state belongs to a mixer of another configuration")
        B, T, _ = x.shape
        if state.carries and state.batch != B:
            raise ValueError(f"the state holds {state.batch} sequences; the input has {B}")
        for t in state._tensors():
            if t.device != x.device:
                raise ValueError(f"the state lives on {t.device}; the input on {x.device} (use state.to)")
        carry = stream.Carry(state.carries, state.position)
        with stream.carrying(carry):
            if T == 0:
                return x.new_empty(B, 0, self.cfg.d_model), state
            memory = carry.take()
            y, memory = self._mix(x, memory, memory if stream.updates_in_place() else None, None, True)
        return y, ThetaScanState(fingerprint=state.fingerprint, position=state.position + T, batch=B, carries=(memory,))

    def _mix(self, x, memory, memory_out, lengths, carried: bool = False):
        cfg = self.cfg
        B, T, D = x.shape
        d = cfg.head_dim

        def heads(lin, width):
            return _linear(x, lin).view(B, T, -1, width).transpose(1, 2)

        q, k = _l2norm(heads(self.proj_q, d)), _l2norm(heads(self.proj_k, d))
        beta, decay = torch.sigmoid(heads(self.beta.lin, 1)), -F.softplus(heads(self.decay.g.lin, 1))
        y = gated_delta_rule(q, k, heads(self.proj_v, d), beta, decay, state=memory, lengths=lengths,
                             return_state=carried, state_out=memory_out)
        y, memory = y if carried else (y, None)
        y = rownorm.rms_rows(y) if rownorm.supported(y) else F.rms_norm(y, (d,))
        y = y * F.silu(heads(self.ogate.g.lin, d))
        return _linear(y.transpose(1, 2).reshape(B, T, D), self.proj_out), memory
