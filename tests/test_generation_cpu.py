"""The hybrid LM's window, sinks and generation: what it refuses (CPU)."""
from __future__ import annotations

import pytest
import torch

from thetascan_amd import hybrid_lm as lm


def test_a_window_adds_no_parameters():
    plain, windowed = lm.HybridLM(), lm.HybridLM(window=64, sinks=4)
    assert lm.parameter_count(plain) == lm.parameter_count(windowed)
    assert plain.state_dict().keys() == windowed.state_dict().keys()
    assert {b.attn.window for b in windowed.blocks if not b.theta} == {64}


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=2.5), dict(window=True), dict(sinks=-1), dict(sinks=1.0)])
def test_windows_that_are_none(kw):
    with pytest.raises(ValueError, match="must be a whole number"):
        lm.HybridLM(**kw)


def test_generation_refuses():
    idx, u = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4)
    with pytest.raises(ValueError, match="needs a model with a window"):
        lm.HybridLM().generate(idx, u)
    model = lm.HybridLM(window=8)
    for bad in ((idx[:1], u), (idx[0], u), (idx[:, :0], u), (idx, u[0])):
        with pytest.raises(ValueError, match="prompts"):
            model.generate(*bad)
