"""A value that is not finite reaches no token before its own, in any form: the outputs
before it are the bits of the call without it."""
from __future__ import annotations

import pytest
import torch

from tests.test_delta_gpu import BF, F32, inputs, on_gpu

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "beta", "decay")
NAN, INF = float("nan"), float("inf")


def run(s, grad=False):
    import thetascan_amd as ts

    leaf = {n: s[n].detach().clone().requires_grad_(grad) for n in NAMES}
    out, S = ts.gated_delta_rule(*leaf.values(), state=s["state"], return_state=True)
    if not grad:
        return out, S
    up = torch.randn(out.shape, generator=torch.Generator(out.device).manual_seed(5), device=out.device).to(out.dtype)
    return out.detach(), S.detach(), *torch.autograd.grad(out, [leaf["q"], leaf["v"]], up)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,dk,f", [(9, 64, 4), (150, 64, 0), (150, 64, 17), (150, 64, 63), (150, 64, 64), (150, 128, 100),
                                    (150, 40, 149), (1100, 64, 700)])
@pytest.mark.parametrize("name,value", [("q", NAN), ("k", NAN), ("k", INF), ("v", NAN), ("v", -INF), ("beta", NAN),
                                        ("beta", INF), ("decay", NAN), ("decay", INF)])
def test_nothing_reaches_earlier_tokens(cuda, name, value, T, dk, f, dtype):
    s = on_gpu(inputs(1, 2, 2, T, dk, 48, dtype, seed=T + f, state=True), cuda, False)
    want, S = run(s)
    s[name] = s[name].clone()
    if s[name].ndim == 4:
        s[name][0, 1, f, 5] = value
    else:
        s[name][0, 1, f] = value
    out, got = run(s)
    # the other head and the tokens before
    assert torch.equal(out[:, 0], want[:, 0]) and torch.equal(got[:, 0], S[:, 0])
    assert torch.equal(out[0, 1, :f], want[0, 1, :f])
    out, want, got, S = out[0, 1, f:], want[0, 1, f:], got[0, 1], S[0, 1]
    if name == "q":  # its own output alone
        assert not bool(out[0].isfinite().any())
        assert torch.equal(out[1:], want[1:]) and torch.equal(got, S)
    elif name == "v":  # its own column alone
        rest = torch.arange(48, device=cuda) != 5
        assert torch.equal(out[:, rest], want[:, rest]) and torch.equal(got[:, rest], S[:, rest])
        assert not bool(out[:, 5].isfinite().any()) and not bool(got[:, 5].isfinite().any())
    else:
        assert not bool(out.isfinite().any()) and not bool(got.isfinite().any())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,f", [(150, 17), (150, 100), (1100, 700)])
def test_gradients_beside_a_value_that_is_not_finite(cuda, T, f, dtype):
    """The values' own gradients do not depend on them; the queries' before it are as
    without it, from it on there are none."""
    s = on_gpu(inputs(1, 1, 1, T, 64, 48, dtype, seed=T + f, state=True), cuda, False)
    want = run(s, True)
    s["v"] = s["v"].clone()
    s["v"][0, 0, f, 5] = NAN
    got = run(s, True)
    assert torch.equal(got[3], want[3])
    assert torch.equal(got[2][0, 0, :f], want[2][0, 0, :f])
    assert not bool(got[2][0, 0, f:].isfinite().any())
