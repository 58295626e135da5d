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


@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_forwards_gradient_is_a_saved_tensor(cuda, dtype):
    """Offloaded with the others, and not kept by a checkpointed loss."""
    import thetascan_amd as ts
    from torch.utils.checkpoint import checkpoint

    z, args, w = some_rows(cuda, 300, 5003, dtype)

    def loss_of(x):
        return ts.policy_loss(x, *args, weights=w, softcap=30.0)[0]

    want = torch.autograd.grad(loss_of(z), z)[0]
    sizes = []

    def pack(x):
        sizes.append(x.numel())
        return x.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda x: x.to(cuda)):
        loss = loss_of(z)
    assert sizes.count(z.numel()) == 2  # the logits and their gradient
    for up in (1.0, 0.3):
        got = torch.autograd.grad(loss, z, torch.tensor(up, device=cuda), retain_graph=True)[0]
        assert torch.equal(got, want if up == 1.0 else torch.autograd.grad(loss_of(z) * up, z)[0])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = checkpoint(loss_of, z, use_reentrant=False)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before < z.numel() * z.element_size() // 2
    assert torch.equal(torch.autograd.grad(loss, z)[0], want)


def test_a_gradient_changed_by_its_owner(cuda):
    """What is done to the first backward's result changes no later one."""
    import thetascan_amd as ts

    z, args, w = some_rows(cuda, 40, 2500, BF)
    loss, _ = ts.policy_loss(z, *args, weights=w)
    first = torch.autograd.grad(loss, z, retain_graph=True)[0]
    held = first.clone()
    first.mul_(2.0)
    assert torch.equal(torch.autograd.grad(loss, z, retain_graph=True)[0], held)
    loss.backward(retain_graph=True)
    loss.backward()
    assert torch.equal(z.grad, held + held)
