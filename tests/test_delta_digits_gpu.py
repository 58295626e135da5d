"""The digits of the gated delta rule's gradients, where sums over alike keys cancel.

Bars, from float64 autograd of the token recurrence.  A bf16 call's products take
operands that are inputs (exact) or bf16 pairs: two roundings of at most 2^-8, the
second of what the first leaves, and the remainders' own product left out, 3 x 2^-16
a product.  Ten of them follow one another at most (state, written rows, their
gradients, pair matrices, the states' gradients, the result): 2^-11 before the result
is rounded, in the 2-norm of a gradient, and of every token's row of it beside the
larger of its own and the rows' mean.  A bf16 gradient is rounded once more, by at
most 2^-8; gates and states in fp32 have only the first.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_delta_gpu import BF, inputs, on_gpu, reference

pytestmark = pytest.mark.gpu

HELD = 2.0 ** -11


def alike(kind, beta, T, decay, dk=64, dv=64, H=2, seed=0):
    """bf16 streams and fp32 gates; keys of one direction ("one"), nearly ("near") or
    half ("half") alike."""
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    q, k = normal(1, H, T, dk), normal(1, H, T, dk)
    first = k[:, :, :1]
    k = {"one": first.expand_as(k), "near": first + 0.1 * k, "half": first + k}[kind]
    q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    lost = torch.nn.functional.softplus(normal(1, H, T) - 3.0) if decay else torch.full((1, H, T), 1e-3)
    return dict(q=q.to(BF), k=k.to(BF), v=normal(1, H, T, dv).to(BF), beta=torch.full((1, H, T), beta),
                decay=-lost, state=0.3 * normal(1, H, dk, dv))


def hold(s, cuda, lengths=None):
    import thetascan_amd as ts

    ref_in = {n: x.double().requires_grad_() for n, x in s.items()}
    ref = reference(**ref_in, lengths=lengths)
    dev = on_gpu(s, cuda, True)
    got = ts.gated_delta_rule(dev["q"], dev["k"], dev["v"], dev["beta"], dev["decay"], state=dev["state"],
                              lengths=None if lengths is None else lengths.to(cuda), return_state=True)
    g = torch.Generator().manual_seed(99)
    up = [torch.randn(ref[0].shape, generator=g).to(s["q"].dtype), torch.randn(ref[1].shape, generator=g)]
    want = torch.autograd.grad(ref, list(ref_in.values()), [x.double() for x in up])
    grads = torch.autograd.grad(got, list(dev.values()), [x.to(cuda) for x in up])
    worst = {}
    for n, w, x in zip(["out", "new state", *s], [*ref, *want], [*got, *grads]):
        bar = HELD + (2.0 ** -8 if x.dtype == BF else 0.0)
        w, x = w.detach(), x.detach().double().cpu()
        whole = float((x - w).norm() / w.norm())
        # a token's row (a gate: one number; a state: a key's)
        rows = w.norm(dim=-1) if w.ndim == 4 else w.abs()
        off = (x - w).norm(dim=-1) if w.ndim == 4 else (x - w).abs()
        row = float((off / rows.clamp_min(float(rows.square().mean().sqrt()))).max())
        worst[n] = (whole, row, bar)
    print(" ".join(f"{n} {a:.1e}/{b:.1e}" for n, (a, b, _) in worst.items()), flush=True)
    bad = {n: x for n, x in worst.items() if not max(x[:2]) <= x[2]}
    assert not bad, bad


@pytest.mark.parametrize("kind,beta,decay", [("near", 1.0, False), ("one", 0.5, False), ("one", 0.9, False),
                                             ("one", 0.9, True), ("one", 1.0, True), ("half", 2.0, False)])
def test_alike_keys_keep_their_digits(cuda, kind, beta, decay):
    hold(alike(kind, beta, 190, decay), cuda)


@pytest.mark.parametrize("dk,dv", [(128, 128), (40, 72), (16, 200)])
def test_widths_keep_their_digits(cuda, dk, dv):
    hold(alike("near", 0.9, 130, True, dk, dv, H=1, seed=dk), cuda)


@pytest.mark.parametrize("Hk,T,dk,lengths", [(2, 150, 64, [150, 70]), (1, 200, 64, None), (1, 1100, 64, [1100, 641]),
                                             (1, 1100, 128, None)])
def test_rows_of_ordinary_keys(cuda, Hk, T, dk, lengths):
    """Every token's row, shared heads, ragged batches and segments of long sequences."""
    s = inputs(2, Hk, 2, T, dk, 64, BF, seed=T, state=True)
    s["beta"], s["decay"] = s["beta"].float(), s["decay"].float() * 0.1
    if lengths:
        for b, n in enumerate(lengths):
            for name in ("q", "k", "v", "beta", "decay"):
                s[name][b, :, n:] = 0.0
        lengths = torch.tensor(lengths)
    hold(s, cuda, lengths)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("H,T", [(2, 2), (2, 70), (1, 200)])
def test_retentions_that_act_on_nothing_have_no_gradient(cuda, H, T, dtype):
    """A first token's without an entering state, and a reset's (-inf, or a factor that
    fp32 does not hold): exactly zero, not what rounding leaves of terms that cancel.
    The others' are as their definition has them."""
    import thetascan_amd as ts

    s = inputs(2, 1, H, T, 64, 40, dtype, seed=T)
    s["beta"], s["decay"] = s["beta"].float(), s["decay"].float()
    resets = [t for t in (1, 40, 64, 65, 130, T - 1) if t < T]
    s["decay"][..., resets] = -float("inf")
    s["decay"][..., resets[-1:]] = -200.0
    del s["state"]
    ref_in = {n: x.double().requires_grad_() for n, x in s.items()}
    ref = sum((x * (i + 1)).sum() for i, x in enumerate(reference(**ref_in)))
    (want,) = torch.autograd.grad(ref, ref_in["decay"])
    dev = on_gpu(s, cuda, True)
    got = ts.gated_delta_rule(*dev.values(), return_state=True)
    (grad,) = torch.autograd.grad(sum((x.float() * (i + 1)).sum() for i, x in enumerate(got)), dev["decay"])
    zero = torch.zeros(T, dtype=torch.bool)
    zero[[0, *resets]] = True
    assert not bool(grad[..., zero].any())
    if T > 2:
        rest = want[..., ~zero]
        assert float((grad.double().cpu()[..., ~zero] - rest).norm()) <= HELD * float(rest.norm())


@pytest.mark.parametrize("Hk,T,dk,dv,lengths", [(2, 200, 64, 64, None), (1, 130, 40, 72, [130, 64]),
                                                (1, 2200, 64, 64, [2200, 1283]), (1, 1100, 128, 128, None)])
def test_states_of_bf16_streams_are_fp32_ones(cuda, Hk, T, dk, dv, lengths):
    """The fp32 state of a bf16 call: operands in three parts hold 24 bits, and what is
    left out of their products is less; some 16 roundings of 2^-24 (the sums of a chunk,
    of the inverse, of what is written and of the state) do not cancel for ordinary keys."""
    import thetascan_amd as ts

    s = inputs(2, Hk, 2, T, dk, dv, BF, seed=T, state=True)
    s["beta"], s["decay"] = s["beta"].float(), s["decay"].float() * 0.1
    if lengths:
        for b, n in enumerate(lengths):
            for name in ("q", "k", "v", "beta", "decay"):
                s[name][b, :, n:] = 0.0
        lengths = torch.tensor(lengths)
    _, want = reference(**s, lengths=lengths)
    dev = on_gpu(s, cuda, False)
    for grad in (False, True):
        q = dev["q"].detach().requires_grad_(grad)
        _, got = ts.gated_delta_rule(q, *(dev[n] for n in ("k", "v", "beta", "decay")), state=dev["state"],
                                     lengths=None if lengths is None else lengths.to(cuda), return_state=True)
        off = float((got.detach().double().cpu() - want).norm() / want.norm())
        print(f"{off:.1e}", flush=True)
        assert off <= 16 * 2.0 ** -24
