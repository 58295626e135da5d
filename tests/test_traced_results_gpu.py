"""The custom ops' results have the shapes, strides and dtypes that their fakes
promise to a compiler, with odd widths, states and every optional input."""
from __future__ import annotations

import pytest
import torch

from tests.test_delta_gpu import BF, F32, inputs, on_gpu

pytestmark = pytest.mark.gpu


def as_promised(op, args):
    torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))
    return op(*args)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("decay", ["token", "head", None])
@pytest.mark.parametrize("dk,dv,T", [(5, 3, 70), (40, 36, 70), (64, 64, 3)])
def test_delta_rule(cuda, dk, dv, T, decay, dtype):
    from thetascan_amd._core.ops import delta

    op = delta._delta_op
    for state in (True, False):
        s = on_gpu(inputs(2, 1, 2, T, dk, dv, dtype, seed=T, decay=decay, state=state), cuda, False)
        first = [s[n] for n in ("q", "k", "v", "beta", "decay", "state")]
        lengths = torch.tensor([T, T // 2], device=cuda)
        for want_state, keep, step in ((True, True, False), (False, False, T < 12)):
            out, final, saved = as_promised(op.op, (*first, lengths, want_state, keep, step))
        out, final, saved = op.op(*first, lengths, True, True, False)
        for up in ((out, final), (out, None), (None, final)):
            as_promised(op.bwd_op, (*up, *first, lengths, saved, state))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [77, 2500])
def test_policy_loss(cuda, V, dtype):
    from thetascan_amd._core.ops import policy

    z = torch.randn(6, V, device=cuda).to(dtype)
    tokens = torch.arange(6, device=cuda)
    rows = torch.zeros(6, device=cuda)
    loss, _, saved = as_promised(policy._policy_op.op, (z, tokens, rows - 3.0, rows + 1.0, rows, None, 0.2, 0.2, 0.1, 30.0))
    as_promised(policy._policy_op.bwd_op, (loss, z, tokens, None, saved, 30.0))
