"""A state that is written in place counts as changed: a recorded graph that saved
its old values refuses its backward, as after torch's own in-place operations."""
from __future__ import annotations

import pytest
import torch

from tests.test_delta_gpu import BF, inputs, on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("dk,dv", [(64, 64), (60, 64)])
def test_a_graph_that_saved_the_old_state_refuses(cuda, T, dk, dv):
    import thetascan_amd as ts

    s = on_gpu(inputs(1, 1, 2, T, dk, dv, BF, seed=T, state=True), cuda, False)
    args = [s[n] for n in ("q", "k", "v", "beta", "decay")]
    S = s["state"].clone().requires_grad_()
    loss = S.square().sum()
    held = S.detach()
    before = held._version
    with torch.no_grad():
        ts.gated_delta_rule(*args, state=held, state_out=held)
    assert held._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # a call without state_out changes nothing it is given
    before = held._version
    with torch.no_grad():
        ts.gated_delta_rule(*args, state=held, return_state=True)
    assert held._version == before


def test_states_of_inference_mode(cuda):
    import thetascan_amd as ts

    s = on_gpu(inputs(1, 1, 2, 3, 64, 64, BF, seed=1, state=True), cuda, False)
    args = [s[n] for n in ("q", "k", "v", "beta", "decay")]
    want, S = ts.gated_delta_rule(*args, state=s["state"], return_state=True)
    with torch.inference_mode():
        held = s["state"].clone()
        out, got = ts.gated_delta_rule(*args, state=held, state_out=held, return_state=True)
    assert got is held and torch.equal(held, S) and torch.equal(out, want)


def test_a_new_state_that_overlaps_the_old_one_is_refused(cuda):
    import thetascan_amd as ts

    s = on_gpu(inputs(2, 1, 2, 3, 64, 64, BF, seed=1), cuda, False)
    args = [s[n] for n in ("q", "k", "v", "beta", "decay")]
    both = torch.zeros(5, 2, 64, 64, device=cuda)
    for old, new in ((both[:2], both[1:3]), (both[2:4], both[1:3])):
        with pytest.raises(ValueError, match="overlaps"):
            ts.gated_delta_rule(*args, state=old, state_out=new)
    assert not bool(both.any())
    # side by side, and the transpose of its own memory (read from a copy)
    ts.gated_delta_rule(*args, state=both[:2], state_out=both[2:4])
    want = ts.gated_delta_rule(*args, state=both[2:4].transpose(2, 3), return_state=True)[1]
    got = ts.gated_delta_rule(*args, state=both[2:4].transpose(2, 3), state_out=both[2:4], return_state=True)[1]
    assert torch.equal(got, want) and got.data_ptr() == both[2:4].data_ptr()
