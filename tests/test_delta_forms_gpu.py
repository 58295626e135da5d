"""Forms of the gated delta rule that the other tests leave out: static retentions in
bf16, the widest values, a second backward, padding that holds NaN behind sequences
cut into segments, compiled calls with a state, and streams past 32-bit offsets."""
from __future__ import annotations

import pytest
import torch

from tests.test_delta_digits_gpu import hold
from tests.test_delta_gpu import BF, F32, OUT, STATE, check, inputs, on_gpu, reference, rel

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "beta", "decay")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,ragged", [(100, False), (450, True)])
def test_static_retentions_in_bf16(cuda, T, ragged, dtype):
    s = inputs(3, 1, 2, T, 64, 48, dtype, seed=T, decay="head", state=True)
    s["decay"] = s["decay"].to(BF)
    lengths = torch.tensor([T, 70, 0]) if ragged else None
    if ragged:
        for b, n in enumerate(lengths.tolist()):
            for name in ("q", "k", "v", "beta"):
                s[name][b, :, n:] = 0.0
    hold(s, cuda, lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dk", [16, 128])
def test_widest_values(cuda, dk, dtype):
    import thetascan_amd as ts
    from thetascan_amd import _lib

    check(inputs(1, 1, 2, 70, dk, 512, dtype, seed=dk, state=True), cuda)
    s = inputs(2, 1, 2, 3, dk, 512, dtype, seed=dk, state=True)
    dev = on_gpu(s, cuda, False)
    want, S = reference(**s)
    with _lib.record_launches() as recs:
        out, got = ts.gated_delta_rule(*(dev[n] for n in NAMES), state=dev["state"], return_state=True)
    assert [r[0] for r in recs] == ["ts_delta_step"]
    assert rel(out, want) <= OUT[dtype] and rel(got, S) <= STATE[dtype]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hk,T,decay", [(1, 100, "token"), (2, 1100, "head")])
def test_a_second_backward_gives_the_same_bits(cuda, Hk, T, decay, dtype):
    import thetascan_amd as ts

    s = on_gpu(inputs(1, Hk, 2, T, 64, 64, dtype, seed=T, decay=decay, state=True), cuda, True)
    out, S = ts.gated_delta_rule(*(s[n] for n in NAMES), state=s["state"], return_state=True)
    ends = [out.detach(), S.detach()]
    first = torch.autograd.grad([out, S], list(s.values()), ends, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad([out, S], list(s.values()), ends)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,dk,dv", [(1537, 64, 40), (2200, 128, 72)])
def test_segments_never_read_behind_a_length(cuda, T, dk, dv, dtype):
    """NaN in every stream and upstream gradient behind the lengths: the bits of zeros."""
    import thetascan_amd as ts

    s = on_gpu(inputs(4, 1, 2, T, dk, dv, dtype, seed=T, state=True), cuda, False)
    lengths = torch.tensor([T, 0, T // 2 + 3, 64], device=cuda)
    past = (torch.arange(T, device=cuda) >= lengths[:, None])[:, None]
    up = torch.randn(4, 2, T, dv, device=cuda).to(dtype)
    dS = torch.randn(4, 2, dk, dv, device=cuda)

    def run(fill):
        leaf = {n: s[n].masked_fill(past if s[n].ndim == 3 else past[..., None], fill).requires_grad_() for n in NAMES}
        leaf["state"] = s["state"].clone().requires_grad_()
        out, S = ts.gated_delta_rule(*(leaf[n] for n in NAMES), state=leaf["state"], lengths=lengths, return_state=True)
        ends = [up.masked_fill(past[..., None], fill), dS]
        return [out.detach(), S.detach(), *torch.autograd.grad([out, S], list(leaf.values()), ends)]

    for a, b in zip(run(float("nan")), run(0.0)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dk,dv", [(5, 3), (40, 36), (64, 64)])
def test_compiled_training_with_a_state(cuda, dk, dv):
    import thetascan_amd as ts

    s = on_gpu(inputs(1, 1, 2, 80, dk, dv, BF, seed=dk, state=True), cuda, True)

    def f(q, k, v, beta, decay, state):
        out, S = ts.gated_delta_rule(q, k, v, beta, decay, state=state, return_state=True)
        return out * 2.0, S * 2.0

    args = list(s.values())
    want, got = f(*args), torch.compile(f, backend="aot_eager", fullgraph=True)(*args)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for a, b in zip(*(torch.autograd.grad([x[0].float().sum(), x[1].sum()], args) for x in (want, got))):
        assert torch.equal(a, b) and a.stride() == b.stride()


def test_many_sequences_of_one_token(cuda):
    import thetascan_amd as ts

    s = on_gpu(inputs(5000, 1, 2, 1, 16, 16, BF, seed=1, state=True), cuda, True)
    args = [s[n] for n in NAMES]
    out, S = ts.gated_delta_rule(*args, state=s["state"], return_state=True)
    with torch.no_grad():
        step, S1 = ts.gated_delta_rule(*args, state=s["state"], return_state=True)
    assert rel(out, step) <= 2 * OUT[BF] and rel(S, S1) <= STATE[BF]
    # out = S'^T q, so a token's value gradient is beta (k . q) times the output's
    (dv,) = torch.autograd.grad(out.float().sum(), s["v"])
    kq = (s["k"].float() * s["q"].float()).sum(-1, keepdim=True)
    assert rel(dv, (s["beta"].float()[..., None] * kq).expand_as(dv)) <= 2.0 ** -8 + 2.0 ** -11


def test_streams_past_32_bit_offsets(cuda):
    """Rows of a [1, 70000, 32768] tensor (2.3e9 elements): the bits of contiguous ones."""
    import thetascan_amd as ts

    T = 70000
    wide = torch.empty(1, T, 32768, dtype=BF, device=cuda)
    s = on_gpu(inputs(1, 1, 1, T, 64, 64, BF, seed=2), cuda, False)
    views = []
    for i, n in enumerate(("q", "k", "v")):
        view = wide[..., 64 * i:64 * i + 64].unsqueeze(1)
        views.append(view.copy_(s[n]).requires_grad_())
    plain = [s[n].contiguous().requires_grad_() for n in ("q", "k", "v")]
    results = []
    for leaves in (views, plain):
        out, S = ts.gated_delta_rule(*leaves, s["beta"], s["decay"], return_state=True)
        results.append([out.detach(), S.detach(), *torch.autograd.grad(out, leaves, out.detach())])
    for a, b in zip(*results):
        assert torch.equal(a, b)
