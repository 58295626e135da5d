"""The policy loss's gradient under upstream gradients that are not one, at both forms
of the backward (rows that leave a gradient in the forward, and rows that do not)."""
from __future__ import annotations

import pytest
import torch

from tests.test_policy_gpu import BF, F32, inputs

pytestmark = pytest.mark.gpu


def some_rows(cuda, N, V, dtype):
    """A loss whose every third row has weight zero and holds nothing."""
    z, tokens, old, ref, adv = inputs(N, V, dtype, seed=V)
    w = torch.rand(N, generator=torch.Generator().manual_seed(1))
    w[::3] = 0.0
    z[::3] = float("nan")
    tokens[::3] = -7
    return z.to(cuda).requires_grad_(), [x.to(cuda) for x in (tokens, old, adv)], w.to(cuda)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V", [(40, 515), (40, 2500), (300, 5003), (6, 70001)])
@pytest.mark.parametrize("upstream", [0.3, -2.5, 1.0, float("inf")])
def test_every_backward_rounds_once_and_leaves_unread_rows_zero(cuda, upstream, N, V, dtype):
    import thetascan_amd as ts

    z, args, w = some_rows(cuda, N, V, dtype)
    loss, _ = ts.policy_loss(z, *args, weights=w, softcap=30.0)
    up = torch.tensor(upstream, device=cuda)
    first = torch.autograd.grad(loss, z, up, retain_graph=True)[0]
    again = torch.autograd.grad(loss, z, up)[0]
    assert torch.equal(first.nan_to_num(), again.nan_to_num()) and torch.equal(first.isnan(), again.isnan())
    assert not bool(first[::3].any())
