"""Gated delta rule (ts_delta_fwd, ts_delta_bwd, ts_delta_step) against the token
recurrence in float64, with autograd's gradients of it.

Bars, in the 2-norm.  A rounding to bf16 is off by at most 2^-8 relative, to
fp32 by 2^-24.  bf16 outputs: one rounding, 2^-8, of sums over operands in bf16
pairs, 2^-16 each (pair matrix, inverse, state, what is written twice).  Gradients: the products of the backward
take up to seven once-rounded operands (pair matrices, written rows, their
gradients, states and their gradients, the inverse) and round the result,
8 x 2^-8.  The state of a bf16 call: five operands in bf16 pairs, 2^-16 each.
fp32: sums of some 200 terms and the exponentials, 2^-24 x 300.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
OUT = {BF: 2.0 ** -8 + 5 * 2.0 ** -16, F32: 300 * 2.0 ** -24}
GRAD = {BF: 8 * 2.0 ** -8, F32: 300 * 2.0 ** -24}
STATE = {BF: 5 * 2.0 ** -16, F32: 300 * 2.0 ** -24}


def reference(q, k, v, beta, decay, state=None, lengths=None):
    """float64, one token after the other; q, k [B,Hk,T,dk], decay a log retention."""
    B, H, T, dv = v.shape
    q, k, v, beta = (x.double() for x in (q, k, v, beta))
    rep = H // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    beta = beta.reshape(B, H, T)
    if decay is None:
        a = torch.ones(B, H, T, dtype=torch.float64)
    elif decay.ndim == 1:
        a = decay.double().exp().view(1, H, 1).expand(B, H, T)
    else:
        a = decay.double().reshape(B, H, T).exp()
    S = torch.zeros(B, H, q.shape[-1], dv, dtype=torch.float64) if state is None else state.double()
    out = []
    for t in range(T):
        A = a[:, :, t, None, None] * S
        u = beta[:, :, t, None] * (v[:, :, t] - (A * k[:, :, t, :, None]).sum(2))
        new = A + k[:, :, t, :, None] * u[:, :, None]
        o = (new * q[:, :, t, :, None]).sum(2)
        if lengths is not None:
            live = (t < lengths).view(B, 1, 1)
            new, o = torch.where(live[..., None], new, S), torch.where(live, o, 0.0)
        S = new
        out.append(o)
    return torch.stack(out, 2), S


def inputs(B, Hk, H, T, dk, dv, dtype, seed=0, decay="token", state=False):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    q, k = normal(B, T, Hk, dk), normal(B, T, Hk, dk)
    k = k + 0.7 * k.roll(1, 1)
    q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    s = dict(q=q, k=k, v=normal(B, T, H, dv))
    s = {n: x.to(dtype).transpose(1, 2) for n, x in s.items()}
    s["beta"] = torch.sigmoid(normal(B, H, T)).to(dtype)
    s["decay"] = None
    if decay == "token":
        s["decay"] = -torch.nn.functional.softplus(normal(B, H, T) - 3.0).to(dtype)
    elif decay == "head":
        s["decay"] = -0.1 * torch.rand(H, generator=g)
    s["state"] = 0.3 * normal(B, H, dk, dv) if state else None
    return s


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def on_gpu(s, cuda, grad):
    return {n: None if x is None else x.to(cuda).requires_grad_(grad) if x.is_floating_point() else x.to(cuda)
            for n, x in s.items()}


def check(s, cuda, lengths=None, grad=True, dtype=None):
    """Outputs, the state and every gradient of one call against the reference."""
    import thetascan_amd as ts

    dtype = dtype or s["q"].dtype
    ref_in = {n: None if x is None else x.double().requires_grad_(grad) for n, x in s.items()}
    ref_out, ref_S = reference(**ref_in, lengths=lengths)
    dev = on_gpu(s, cuda, grad)
    out, S = ts.gated_delta_rule(dev["q"], dev["k"], dev["v"], dev["beta"], dev["decay"], state=dev["state"],
                                 lengths=None if lengths is None else lengths.to(cuda), return_state=True)
    assert out.shape == ref_out.shape and out.dtype == dtype and S.dtype == F32
    errs = {"out": (rel(out, ref_out), OUT[dtype]), "state": (rel(S, ref_S), STATE[dtype])}
    if grad:
        g = torch.Generator().manual_seed(99)
        do = torch.randn(ref_out.shape, generator=g).to(dtype)
        dS = torch.randn(ref_S.shape, generator=g)
        names = [n for n in s if s[n] is not None]
        ref_g = torch.autograd.grad([ref_out, ref_S], [ref_in[n] for n in names], [do.double(), dS.double()])
        got = torch.autograd.grad([out, S], [dev[n] for n in names], [do.to(cuda), dS.to(cuda)])
        for n, r, x in zip(names, ref_g, got):
            assert x.shape == r.shape and x.dtype == s[n].dtype, n
            errs["d" + n] = (rel(x, r), GRAD[dtype])
    print(" ".join(f"{n} {e:.1e}" for n, (e, _) in errs.items()), flush=True)
    bad = {n: e for n, (e, bar) in errs.items() if not e <= bar}
    assert not bad, bad
    return dev, out, S


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 2, 16, 17, 63, 64, 65, 127, 200])
def test_lengths_of_the_sequence(cuda, T, dtype):
    check(inputs(2, 2, 2, T, 64, 64, dtype, seed=T, state=True), cuda)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dk,dv", [(8, 8), (5, 3), (16, 100), (48, 80), (64, 129), (72, 16), (128, 64), (100, 200)])
def test_widths(cuda, dk, dv, dtype):
    check(inputs(1, 2, 2, 90, dk, dv, dtype, seed=dk + dv, state=True), cuda)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hk,H", [(1, 4), (2, 6), (3, 3)])
@pytest.mark.parametrize("decay", ["token", "head", None])
def test_shared_heads_and_retentions(cuda, Hk, H, decay, dtype):
    check(inputs(2, Hk, H, 100, 64, 64, dtype, seed=Hk, decay=decay), cuda)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_padded_batch_never_reads_behind_a_length(cuda, dtype):
    s = inputs(6, 2, 4, 150, 64, 48, dtype, seed=3, state=True)
    lengths = torch.tensor([150, 0, 1, 64, 65, 149])
    for b, n in enumerate(lengths.tolist()):
        for name in ("q", "k", "v", "beta", "decay"):
            s[name][b, :, n:] = 0.0
    # (behind the lengths nothing is read: the call itself gets NaN there)
    dev = {n: x.clone() for n, x in s.items()}
    for b, n in enumerate(lengths.tolist()):
        for name in ("q", "k", "v", "beta", "decay"):
            dev[name][b, :, n:] = float("nan")
    import thetascan_amd as ts

    ref_in = {n: x.double().requires_grad_() for n, x in s.items()}
    ref_out, ref_S = reference(**ref_in, lengths=lengths)
    leaf = on_gpu(dev, cuda, True)
    out, S = ts.gated_delta_rule(leaf["q"], leaf["k"], leaf["v"], leaf["beta"], leaf["decay"], state=leaf["state"],
                                 lengths=lengths.to(cuda), return_state=True)
    g = torch.Generator().manual_seed(1)
    do = torch.randn(ref_out.shape, generator=g).to(dtype)
    names = list(s)
    ref_g = torch.autograd.grad(ref_out, [ref_in[n] for n in names], do.double())
    do_dev = do.clone()
    for b, n in enumerate(lengths.tolist()):
        do_dev[b, :, n:] = float("nan")
    got = torch.autograd.grad(out, [leaf[n] for n in names], do_dev.to(cuda))
    assert rel(out, ref_out) <= OUT[dtype] and rel(S, ref_S) <= STATE[dtype]
    for n, r, x in zip(names, ref_g, got):
        assert bool(torch.isfinite(x).all()), n
        assert rel(x, r) <= GRAD[dtype], (n, rel(x, r))
    for b, n in enumerate(lengths.tolist()):
        assert not bool(out[b, :, n:].any())
        for name, x in zip(names, got):
            if name != "state":
                assert not bool(x[b, :, n:].any()), name
    # a sequence of no tokens: its state is passed on bit for bit
    assert torch.equal(S[1], leaf["state"][1])
    # and the token form agrees
    with torch.no_grad():
        few = {n: x[:, :, :8] if n != "state" else x for n, x in leaf.items()}
        o8, S8 = ts.gated_delta_rule(few["q"], few["k"], few["v"], few["beta"], few["decay"], state=few["state"],
                                     lengths=lengths.to(cuda, torch.int32), return_state=True)
    r8, rS8 = reference(*(s[n][:, :, :8] for n in ("q", "k", "v", "beta", "decay")), s["state"], lengths)
    assert rel(o8, r8) <= OUT[dtype] and rel(S8, rS8) <= 300 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [BF, F32])
def test_write_strength_zero_and_resets(cuda, dtype):
    """beta exactly zero (whose own gradient is not), retentions of -inf and of
    hundreds of nats beside ordinary ones, several of them in one chunk."""
    s = inputs(2, 2, 2, 150, 64, 64, dtype, seed=5, state=True)
    s["beta"][:, :, ::7] = 0.0
    s["beta"][0, 0] = 0.0
    s["decay"][:, :, [3, 4, 40, 90, 140]] = -float("inf")
    s["decay"][:, :, [10, 11, 70, 71]] = -300.0
    check(s, cuda)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_alike_keys(cuda, dtype):
    """One key throughout and full write strength: the triangular system of a
    chunk has every entry at its largest."""
    s = inputs(1, 1, 2, 130, 64, 64, dtype, seed=6, decay=None)
    s["k"] = s["k"][:, :, :1].expand(-1, -1, 130, -1).contiguous()
    s["beta"] = torch.ones_like(s["beta"])
    check(s, cuda, grad=False)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 3, 8])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (40, 36), (5, 3)])
def test_recurrent_form(cuda, T, dk, dv, dtype):
    """Few tokens without gradients: one launch of ts_delta_step, in fp32."""
    import thetascan_amd as ts
    from thetascan_amd import _lib

    s = inputs(3, 2, 4, T, dk, dv, dtype, seed=T + dk, state=True)
    dev = on_gpu(s, cuda, False)
    ref, ref_S = reference(**s)
    with torch.no_grad(), _lib.record_launches() as recs:
        out, S = ts.gated_delta_rule(dev["q"], dev["k"], dev["v"], dev["beta"], dev["decay"], state=dev["state"],
                                     return_state=True)
    assert [r[0] for r in recs] == ["ts_delta_step"]
    assert rel(S, ref_S) <= 300 * 2.0 ** -24
    assert rel(out, ref) <= (2.0 ** -8 if dtype == BF else 300 * 2.0 ** -24)
    # in place, the same numbers
    held = dev["state"].clone()
    out2, S2 = ts.gated_delta_rule(dev["q"], dev["k"], dev["v"], dev["beta"], dev["decay"], state=held, state_out=held,
                                   return_state=True)
    assert S2 is held and torch.equal(held, S) and torch.equal(out2, out)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_pieces_equal_the_whole(cuda, dtype):
    import thetascan_amd as ts

    s = inputs(2, 2, 4, 200, 64, 64, dtype, seed=8)
    dev = on_gpu(s, cuda, False)
    args = [dev[n] for n in ("q", "k", "v", "beta", "decay")]
    whole, S = ts.gated_delta_rule(*args, return_state=True)
    state, outs = None, []
    for a, b in ((0, 70), (70, 71), (71, 79), (79, 200)):
        piece = [x[:, :, a:b] for x in args]
        o, state = ts.gated_delta_rule(*piece, state=state, return_state=True)
        outs.append(o)
    # (each side is off the exact answer by at most the bar)
    assert rel(torch.cat(outs, 2), whole) <= 2 * OUT[dtype]
    assert rel(state, S) <= 2 * STATE[dtype]


def test_strides_and_memory_orders_bit_for_bit(cuda):
    """Rows of wider matrices, head-major and token-major memory, broadcast
    gates, misaligned rows: the same numbers as of contiguous tensors."""
    import thetascan_amd as ts

    s = inputs(2, 2, 2, 100, 64, 64, BF, seed=9)
    dev = on_gpu(s, cuda, False)
    plain = [dev[n].contiguous() for n in ("q", "k", "v", "beta", "decay")]

    def call(args):
        leaves = [x.detach().requires_grad_() for x in args]
        out, S = ts.gated_delta_rule(*leaves, return_state=True)
        return [out.detach(), S.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))]

    want = call(plain)
    wide = torch.randn(2, 100, 3 * 128 + 8, device=cuda).bfloat16()
    rows = [wide[..., i * 128:i * 128 + 128].unflatten(-1, (2, 64)).transpose(1, 2) for i in range(3)]
    odd = [wide[..., i * 128 + 1:i * 128 + 129].unflatten(-1, (2, 64)).transpose(1, 2) for i in range(3)]
    for views in (rows, odd):
        for x, y in zip(views, plain):
            x.copy_(y)
        gates = [g.transpose(1, 2).contiguous().transpose(1, 2).unsqueeze(-1) for g in plain[3:]]
        got = call([*views, *gates])
        got[-2:] = [g.squeeze(-1) for g in got[-2:]]
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    # gates broadcast over heads, an upstream gradient that is one broadcast value
    b1, d1 = (g[:, :1].expand(2, 2, 100) for g in plain[3:])
    for a, b in zip(call([*plain[:3], b1, d1]), call([*plain[:3], b1.contiguous(), d1.contiguous()])):
        assert torch.equal(a, b)


def test_repeated_calls_give_the_same_bits(cuda):
    s = on_gpu(inputs(2, 1, 4, 300, 128, 96, BF, seed=10, state=True), cuda, True)
    import thetascan_amd as ts

    def once():
        out, S = ts.gated_delta_rule(s["q"], s["k"], s["v"], s["beta"], s["decay"], state=s["state"], return_state=True)
        return [out.detach(), S.detach(), *torch.autograd.grad([out, S], list(s.values()), [out.detach(), S.detach()])]

    first = once()
    for _ in range(3):
        for a, b in zip(once(), first):
            assert torch.equal(a, b)


def test_gradients_against_differences(cuda):
    """fp32, a step of 2^-6 along a random direction per input: the central
    difference is off by the third derivative (about the step squared) and by the
    outputs' rounding over the step."""
    import thetascan_amd as ts

    s = on_gpu(inputs(1, 1, 2, 70, 64, 32, F32, seed=11, state=True), cuda, True)
    g = torch.Generator(device=cuda).manual_seed(0)
    names = list(s)
    weight = torch.randn(1, 2, 70, 32, generator=g, device=cuda)

    def loss(p):
        out = ts.gated_delta_rule(p["q"], p["k"], p["v"], p["beta"], p["decay"], state=p["state"])
        return (out.double() * weight).sum()

    grads = dict(zip(names, torch.autograd.grad(loss(s), [s[n] for n in names])))
    h = 2.0 ** -6
    for n in names:
        d = torch.randn(s[n].shape, generator=g, device=cuda)
        d = d / d.norm()
        with torch.no_grad():
            ends = [loss({**s, n: s[n] + e * h * d}) for e in (1, -1)]
        measured = float(ends[0] - ends[1]) / (2 * h)
        want = float((grads[n].double() * d).sum())
        scale = float(grads[n].double().norm())
        print(f"{n}: {measured:.6f} {want:.6f}", flush=True)
        assert abs(measured - want) <= 4 * h * h * max(scale, 1.0), n


def test_graph_replays_follow_the_inputs(cuda):
    """Forward and backward captured, and a step in place on its state; replays
    with eager work between them equal the eager calls."""
    import thetascan_amd as ts

    s = on_gpu(inputs(2, 2, 2, 140, 64, 64, BF, seed=12, decay="head"), cuda, True)
    names = [n for n in s if s[n] is not None]
    do = torch.randn(2, 2, 140, 64, device=cuda).bfloat16()

    def train():
        out = ts.gated_delta_rule(s["q"], s["k"], s["v"], s["beta"], s["decay"])
        return [out, *torch.autograd.grad(out, [s[n] for n in names], do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = train()
    for i in range(4):
        with torch.no_grad():
            for n in names:
                s[n].mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, train()):
            assert torch.equal(a, b)


def test_other_stream_and_empty_sequence(cuda):
    import thetascan_amd as ts

    s = on_gpu(inputs(1, 2, 2, 80, 64, 64, BF, seed=13, state=True), cuda, False)
    args = [s[n] for n in ("q", "k", "v", "beta", "decay")]
    want = ts.gated_delta_rule(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ts.gated_delta_rule(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out, S = ts.gated_delta_rule(*(x[:, :, :0] for x in args), state=s["state"], return_state=True)
    assert out.shape == (1, 2, 0, 64) and torch.equal(S, s["state"]) and S is not s["state"]


@pytest.mark.parametrize("decay", ["token", "head", None])
def test_compiled_call_is_the_eager_one(cuda, decay):
    import thetascan_amd as ts

    s = on_gpu(inputs(1, 2, 2, 80, 64, 64, BF, seed=14, decay=decay), cuda, True)
    args = [s[n] for n in ("q", "k", "v", "beta", "decay") if s[n] is not None]

    def f(*a):
        return ts.gated_delta_rule(*a) * 2.0

    out = f(*args)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*args)
    assert torch.equal(out, got)
    for a, b in zip(torch.autograd.grad(out, args, torch.ones_like(out)),
                    torch.autograd.grad(got, args, torch.ones_like(got))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,dk,dv,ragged", [(1024, 64, 64, False), (1537, 64, 40, True), (2200, 128, 72, True)])
def test_long_sequences_in_segments(cuda, T, dk, dv, ragged, dtype):
    """Sequences whose chunks are cut into segments that run side by side: their
    entering states, the lengths that end in any of them, and the gradients behind."""
    from thetascan_amd._core.ops import delta
    from thetascan_amd import _lib
    import ctypes

    s = inputs(4 if ragged else 1, 1, 2, T, dk, dv, dtype, seed=T, state=True)
    s["decay"] = s["decay"] * 0.05  # (a memory that reaches over the segments)
    lengths = torch.tensor([T, 0, T // 2 + 3, 64]) if ragged else None
    one = delta._desc(*(s[n][:1] for n in ("q", "k", "v", "beta", "decay")), False)
    n, short = ctypes.c_size_t(), ctypes.c_size_t()
    _lib.load().ts_delta_workspace_bytes(ctypes.byref(one), ctypes.byref(n))
    per_chunk = n.value / (2 * -(-T // 64))
    one.T = 64
    _lib.load().ts_delta_workspace_bytes(ctypes.byref(one), ctypes.byref(short))
    assert per_chunk > short.value / 2  # segments' states beside the chunks' records
    if ragged:
        for b, m in enumerate(lengths.tolist()):
            for name in ("q", "k", "v", "beta", "decay"):
                s[name][b, :, m:] = 0.0
    check(s, cuda, lengths=lengths)


@pytest.mark.parametrize("T", [100, 2100])
def test_new_state_in_place_of_the_old(cuda, T):
    """state_out = state, also where segments of the sequence run side by side:
    the numbers of a call with a tensor of its own, whatever the lengths."""
    import thetascan_amd as ts

    s = on_gpu(inputs(5, 1, 2, T, 64, 64, BF, seed=T, state=True), cuda, False)
    args = [s[n] for n in ("q", "k", "v", "beta", "decay")]
    lengths = torch.tensor([T, 0, 1, T - 1, T // 2], device=cuda)
    want, S = ts.gated_delta_rule(*args, state=s["state"], lengths=lengths, return_state=True)
    for _ in range(3):
        held = s["state"].clone()
        out, got = ts.gated_delta_rule(*args, state=held, state_out=held, lengths=lengths, return_state=True)
        assert got is held and torch.equal(held, S) and torch.equal(out, want)
    # into a tensor of its own, without the state's being asked for
    other = torch.full_like(S, float("nan"))
    assert torch.equal(ts.gated_delta_rule(*args, state=s["state"], lengths=lengths, state_out=other), want)
    assert torch.equal(other, S)


def test_traced_calls_of_changing_lengths(cuda):
    import thetascan_amd as ts

    fn = torch.compile(lambda *x: ts.gated_delta_rule(*x, return_state=True), backend="aot_eager", dynamic=True,
                       fullgraph=True)
    for T in (70, 129, 5):
        gen = torch.Generator(cuda).manual_seed(T)
        args = [torch.randn(2, h, T, d, device=cuda, generator=gen).mul(d ** -0.5).requires_grad_()
                for h, d in ((2, 16), (2, 16), (4, 24))]
        args.append(torch.rand(2, 4, T, device=cuda, generator=gen).requires_grad_())
        want, got = ts.gated_delta_rule(*args, return_state=True), fn(*args)
        for a, b in zip(want, got):
            assert torch.equal(a, b)
        for a, b in zip(*(torch.autograd.grad(x[0].sum() + x[1].sum(), args) for x in (want, got))):
            assert torch.equal(a, b)
        with torch.no_grad():
            for a, b in zip(ts.gated_delta_rule(*args, return_state=True), fn(*args)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("T,launch", [(12, "ts_delta_step"), (13, "ts_delta_fwd")])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dk,dv", [(64, 96), (72, 40)])
def test_a_ragged_batch_of_few_tokens(cuda, T, launch, dk, dv, dtype):
    """Both forms at the border between them, with sequences that end before T."""
    import thetascan_amd as ts
    from thetascan_amd import _lib

    s = inputs(3, 2, 4, T, dk, dv, dtype, seed=T + dk, state=True)
    lengths = torch.tensor([T, 5, 0])
    dev = on_gpu(s, cuda, False)
    ref, ref_S = reference(**s, lengths=lengths)
    with torch.no_grad(), _lib.record_launches() as recs:
        out, S = ts.gated_delta_rule(dev["q"], dev["k"], dev["v"], dev["beta"], dev["decay"], state=dev["state"],
                                     lengths=lengths.to(cuda), return_state=True)
    assert [r[0] for r in recs] == [launch]
    assert rel(S, ref_S) <= STATE[dtype] and rel(out, ref) <= OUT[dtype]
    assert torch.equal(S[2], dev["state"][2]) and not out[1, :, 5:].any() and not out[2].any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,dk,dv,ragged", [(1, 385, 64, 64, False), (3, 700, 40, 72, True), (1, 517, 128, 128, False),
                                              (2, 2111, 128, 24, True)])
def test_short_sequences_in_uneven_segments(cuda, B, T, dk, dv, ragged, dtype):
    s = inputs(B, 1, 2, T, dk, dv, dtype, seed=T, state=True)
    s["decay"] = s["decay"] * 0.05
    lengths = torch.tensor([T, T // 2, 129][:B]) if ragged else None
    if ragged:
        for b, m in enumerate(lengths.tolist()):
            for name in ("q", "k", "v", "beta", "decay"):
                s[name][b, :, m:] = 0.0
    check(s, cuda, lengths=lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_first_token_forgets_nothing(cuda, dtype):
    """Without an entering state the first token's retention acts on nothing: its
    gradient is zero, not what rounding leaves of terms that cancel."""
    import thetascan_amd as ts

    for T in (1, 70):
        s = on_gpu(inputs(2, 1, 2, T, 64, 40, dtype, seed=T), cuda, True)
        args = [s[n] for n in ("q", "k", "v", "beta", "decay")]
        out, S = ts.gated_delta_rule(*args, return_state=True)
        (g,) = torch.autograd.grad(out.float().sum() + S.sum(), s["decay"])
        if T == 1:
            assert not g.any()
        else:
            assert g[..., 1:].any()
