"""Forward-mode tangents, which no kernel carries, are refused instead of dropped."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import thetascan_amd as ts
from tests.test_delta_cpu import streams


def test_tangents_are_refused():
    for name in ("q", "k", "v", "beta", "retention", "state"):
        s = streams()
        s.update(retention=torch.zeros(2, 4, 10), state=torch.zeros(2, 4, 16, 8))
        with forward_ad.dual_level():
            s[name] = forward_ad.make_dual(s[name], torch.ones_like(s[name]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ts.gated_delta_rule(**s)
    rows = torch.zeros(5)
    with forward_ad.dual_level():
        z = forward_ad.make_dual(torch.zeros(5, 7), torch.ones(5, 7))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ts.policy_loss(z, rows.long(), rows, rows)
        # (a level alone changes nothing)
        with pytest.raises(RuntimeError, match="must live on the GPU"):
            ts.policy_loss(torch.zeros(5, 7), rows.long(), rows, rows)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: ts.policy_loss(x, rows.long(), rows, rows)[0], (torch.zeros(5, 7),), (torch.ones(5, 7),))
