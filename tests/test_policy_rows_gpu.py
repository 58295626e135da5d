"""Rows of weight zero in every kernel of the policy loss, and logits past 32-bit offsets."""
from __future__ import annotations

import pytest
import torch

from tests.test_policy_gpu import BF, F32, compare, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V", [(200, 515), (40, 5003), (300, 9000), (16389, 257), (6, 70001)])
def test_unread_rows_in_every_form(cuda, N, V, dtype):
    """One wave a row, a workgroup a row (with and without the gradient in the forward),
    eight rows' terms together, and several workgroups a row."""
    import thetascan_amd as ts

    z, tokens, old, ref, adv = inputs(N, V, dtype, seed=V)
    w = torch.rand(N, generator=torch.Generator().manual_seed(1)) / N
    out = torch.zeros(N, dtype=torch.bool)
    out[::3] = True
    w[out] = 0.0
    for x in (z, old, ref, adv):
        x[out] = float("nan")
    z[3] = float("inf")
    tokens[out] = -7
    _, lp, dz = compare(cuda, z, tokens, old, adv, ref, w, (0.1, 0.3), 0.3, 30.0, upstream=-2.5)
    assert not bool(lp[out].any()) and not bool(dz[out].any())
    # without a gradient, and the log-probabilities alone, on the rows that count
    with torch.no_grad():
        loss, again = ts.policy_loss(z.to(cuda), tokens.to(cuda), old.to(cuda), adv.to(cuda), ref_log_probs=ref.to(cuda),
                                     weights=w.to(cuda), clip=(0.1, 0.3), kl=0.3, softcap=30.0)
    assert bool(torch.isfinite(loss)) and not bool(again[out].any())
    assert float((again - lp).abs().max()) <= 2.0 ** -18
    alone = ts.token_log_probs(z[~out].to(cuda), tokens[~out].to(cuda), softcap=30.0)
    assert float((alone - lp[~out]).abs().max()) <= 2.0 ** -18


def test_logits_past_32_bit_offsets(cuda):
    """70000 rows of 32768 (2.3e9 logits): the last rows against float64."""
    import thetascan_amd as ts

    N, V, L = 70000, 32768, 32
    z = torch.randn(N, V, dtype=BF, device=cuda, generator=torch.Generator(cuda).manual_seed(0))
    tokens = torch.randint(0, V, (N,), device=cuda, generator=torch.Generator(cuda).manual_seed(1))
    w = torch.zeros(N, device=cuda)
    w[-L:] = 1.0
    zeros = torch.zeros(N, device=cuda)
    z.requires_grad_()
    loss, lp = ts.policy_loss(z, tokens, zeros - 10.0, zeros + 1.0, weights=w, clip=1.0)
    (dz,) = torch.autograd.grad(loss, z)
    last = z[-L:].detach().double().requires_grad_()
    want = torch.log_softmax(last, -1)[torch.arange(L, device=cuda), tokens[-L:]]
    assert float((lp[-L:].double() - want).abs().max()) <= 2.0 ** -17
    ratio = (want + 10.0).exp()
    total = -torch.minimum(ratio, ratio.clamp(0.0, 2.0)).sum()
    (g,) = torch.autograd.grad(total, last)
    assert abs(float(loss) - float(total)) <= 2.0 ** -16 * float(ratio.sum())
    assert float((dz[-L:].double() - g).norm()) <= 2.0 ** -8 * float(g.norm()) + 2.0 ** -16 * float(ratio.norm())
    assert not bool(dz[:N - L].any())
