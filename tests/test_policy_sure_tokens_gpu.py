"""Tokens that are (nearly) certain under a soft cap: log-probabilities never above zero.

Bar.  A row's sum is one and what the others hold, 1 - p: each of their exponents is
off by two capped logits' errors, cap 2^-22 together, and the sum rounds at one, 2^-24
an addition, V / 64 of them a lane and 8 to join the lanes.  Log-probabilities round
once more, 2^-24 of themselves.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V", [(64, 300), (16400, 300), (40, 5003), (8, 70001)])
@pytest.mark.parametrize("cap", [30.0, 64.0, 100.0, None])
@pytest.mark.parametrize("above", [20.0, 40.0])
def test_log_probabilities_of_sure_tokens(cuda, above, cap, N, V, dtype):
    import thetascan_amd as ts

    g = torch.Generator(cuda).manual_seed(V)
    z = 2.0 * torch.randn(N, V, generator=g, device=cuda)
    tokens = torch.randint(0, V, (N,), generator=g, device=cuda)
    rows = torch.arange(N, device=cuda)
    z[rows, tokens] = above + torch.randn(N, generator=g, device=cuda)
    z = z.to(dtype)
    y = cap * torch.tanh(z.double() / cap) if cap else z.double()
    want = torch.log_softmax(y, -1)[rows, tokens]
    other = -torch.expm1(want)
    bar = other * (cap or 1.0) * 2.0 ** -22 + (V / 64 + 8) * 2.0 ** -24 + want.abs() * 2.0 ** -24
    zd = z.requires_grad_()
    _, seen = ts.policy_loss(zd, tokens, want.float(), torch.ones(N, device=cuda), softcap=cap)
    for lp in (ts.token_log_probs(z, tokens, softcap=cap), seen):
        assert float(lp.max()) <= 0.0
        assert bool(((lp.double() - want).abs() <= bar).all())
