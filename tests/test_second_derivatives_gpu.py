"""Gradients that are asked for with create_graph are the ordinary ones, and refuse to
be differentiated again instead of counting as constants."""
from __future__ import annotations

import pytest
import torch

from tests.test_delta_gpu import F32, inputs, on_gpu

pytestmark = pytest.mark.gpu


def refuses(loss, leaf):
    (want,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (grad,) = torch.autograd.grad(loss, leaf, create_graph=True)
    assert torch.equal(grad, want)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (grad.square().sum() + leaf.square().sum()).backward()


def test_delta_rule(cuda):
    import thetascan_amd as ts

    s = on_gpu(inputs(1, 1, 2, 40, 64, 64, F32, seed=1, state=True), cuda, True)
    out, S = ts.gated_delta_rule(*(s[n] for n in ("q", "k", "v", "beta", "decay")), state=s["state"], return_state=True)
    refuses(out.square().sum() + S.sum(), s["k"])


@pytest.mark.parametrize("V", [64, 2500])
def test_policy_loss(cuda, V):
    import thetascan_amd as ts

    z = torch.randn(5, V, device=cuda, requires_grad=True)
    rows = torch.zeros(5, device=cuda)
    refuses(ts.policy_loss(z, rows.long(), rows - 4.0, rows + 1.0)[0], z)
