"""Capped logits as fp32 holds them, whatever the cap.

Bars.  The capped logit is rounded once or twice, 2^-23 of itself: a row's sum is off by
that of its largest ones, |y| 2^-23; the exponents' products by log2 e, 2^-24 of the few
units between those; the exponential and a lane's sum some 2^-23 each, five of them; the
result rounds, 2^-24 of itself.  A saturated logit's slope 4 r (1 - r), r = 1 / (1 + e^x):
x = 2 |z| / cap is rounded twice and the exponential of it is off by as much, then three
roundings: (2 x + 4) 2^-23 of it.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_policy_gpu import BF, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [300, 5003, 70001])
@pytest.mark.parametrize("cap", [20.0, 30.0, 64.0, 200.0])
def test_log_probabilities_do_not_lose_digits_to_the_cap(cuda, cap, V, dtype):
    import thetascan_amd as ts

    N = 8 if V == 70001 else 400
    g = torch.Generator(cuda).manual_seed(V)
    z = (2.0 * torch.randn(N, V, generator=g, device=cuda)).to(dtype)
    tokens = torch.randint(0, V, (N,), generator=g, device=cuda)
    y = cap * torch.tanh(z.double() / cap)
    want = torch.log_softmax(y, -1).gather(-1, tokens[:, None])[:, 0]
    bar = y.abs().amax(-1) * 2.0 ** -23 + 5 * 2.0 ** -23 + want.abs() * 2.0 ** -24
    off = (ts.token_log_probs(z, tokens, softcap=cap).double() - want).abs()
    print(f"{float(off.max()):.1e} {float((off / bar).max()):.2f}", flush=True)
    assert bool((off <= bar).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [300, 5003])
@pytest.mark.parametrize("at", [0.4, 0.6, 2.0, 5.0, 8.0, 12.0])
def test_slopes_of_saturated_logits(cuda, at, V, dtype):
    """Each sign of a token's logit at a multiple of the cap, in whole and in mixed vectors."""
    import thetascan_amd as ts

    N, cap = 32, 30.0
    z = torch.randn(N, V, generator=torch.Generator().manual_seed(0)).to(dtype)
    tokens = torch.arange(N)
    z[torch.arange(N), tokens] = at * cap * (1.0 - 2.0 * (torch.arange(N) % 2)).to(dtype)
    old = torch.full((N,), -3.0)
    zr = z.double().requires_grad_()
    y = cap * torch.tanh(zr / cap)
    lp = torch.log_softmax(y, -1)[torch.arange(N), tokens]
    # (ratios without a border, so that every token has its gradient; the slope in exact form)
    w = (lp + 3.0).exp().detach() / N
    x = 2.0 * z.double().abs() / cap
    r = 1.0 / (1.0 + x.exp())
    p = torch.softmax(y.detach(), -1)
    tok = torch.zeros_like(p).scatter_(1, tokens[:, None], 1.0)
    want = (-w[:, None] * (tok - p) * 4.0 * r * (1.0 - r))[torch.arange(N), tokens]
    zd = z.to(cuda).requires_grad_()
    loss, _ = ts.policy_loss(zd, tokens.to(cuda), old.to(cuda), torch.ones(N, device=cuda), clip=(0.2, 1e30), softcap=cap)
    (dz,) = torch.autograd.grad(loss, zd)
    got = dz[torch.arange(N), tokens].double().cpu()
    rest = (1.0 - p)[torch.arange(N), tokens]
    # (1 - p is off by p's own rounding where p is nearly one; the ratio by 2^-16)
    bar = (2.0 ** -16 + (4.0 * at + 4.0) * 2.0 ** -23 + 2.0 ** -20 / rest.clamp_min(1e-30)
           + (2.0 ** -8 if dtype == BF else 0.0))
    off = (got - want).abs() / want.abs()
    assert bool((off <= bar).all()), float((off / bar).max())
