"""Clipped policy loss (ts_policy_loss_fwd / ts_policy_loss_bwd) against its
definition in float64 with autograd.

Bars.  Log-probabilities: fp32 sums of V exponentials of arguments rounded at
30 log2 e (absolute 2^-19 each with a cap of 30, independent in the sum) and the
result's rounding: 2^-17 absolute.  Loss: exp of that, 2^-16 relative to the sum of
the terms' sizes.  The logits' gradient is dloss/dlp (1[v = token] - p_v): p is off
by 2^-16 of itself, so a row is off by 2^-16 |dloss/dlp| (which is all that is left
where p of the token is 1 and the difference cancels); bf16 rounds it once, 2^-8.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def reference(z, tokens, old, adv, ref=None, weights=None, clip=(0.2, 0.2), kl=0.0, cap=None):
    z, old, adv = z.double(), old.double(), adv.double()
    w = torch.full(old.shape, 1.0 / max(old.numel(), 1), dtype=torch.float64) if weights is None else weights.double()
    on = w != 0
    z = torch.where(on[:, None], z, 0.0)
    y = cap * torch.tanh(z / cap) if cap else z
    lp = torch.log_softmax(y, -1).gather(-1, tokens.clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    lp = torch.where(on, lp, 0.0)
    r = torch.where(on, lp - old, 0.0).exp()
    adv = torch.where(on, adv, 0.0)
    each = -torch.minimum(r * adv, r.clamp(1 - clip[0], 1 + clip[1]) * adv)
    if kl:
        d = torch.where(on, ref.double() - lp, 0.0)
        each = each + kl * (d.exp() - d - 1)
    return (w * each).sum(), lp, (w * each).abs().sum()


def inputs(N, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = (3.0 * torch.randn(N, V, generator=g)).to(dtype)
    tokens = torch.randint(0, V, (N,), generator=g)
    lp = torch.log_softmax(z.double(), -1).gather(-1, tokens[:, None])[:, 0]
    old = (lp + 0.4 * torch.randn(N, generator=g).double()).float()
    ref = (lp + 0.4 * torch.randn(N, generator=g).double()).float()
    adv = torch.randn(N, generator=g)
    return z, tokens, old, ref, adv


def compare(cuda, z, tokens, old, adv, ref=None, weights=None, clip=(0.2, 0.2), kl=0.0, cap=None, upstream=1.0):
    import thetascan_amd as ts

    zr = z.double().requires_grad_()
    want, lp_want, scale = reference(zr, tokens, old, adv, ref, weights, clip, kl, cap)
    dz_want, dlp = torch.autograd.grad(want * upstream, (zr, lp_want))
    zd = z.to(cuda).requires_grad_()
    opt = {n: None if x is None else x.to(cuda) for n, x in (("ref_log_probs", ref), ("weights", weights))}
    loss, lp = ts.policy_loss(zd, tokens.to(cuda), old.to(cuda), adv.to(cuda), **opt, clip=clip, kl=kl, softcap=cap)
    assert loss.dtype == F32 and loss.shape == () and lp.dtype == F32 and not lp.requires_grad
    (dz,) = torch.autograd.grad(loss * upstream, zd)
    assert dz.dtype == z.dtype and dz.shape == z.shape
    lp_err = float((lp.double().cpu() - lp_want).abs().max())
    loss_err = abs(float(loss) - float(want)) / max(float(scale), 1e-30)
    dz_err = float((dz.double().cpu() - dz_want).norm())
    print(f"lp {lp_err:.1e} loss {loss_err:.1e} dz {dz_err:.1e}", flush=True)
    assert lp_err <= 2.0 ** -17 and loss_err <= 2.0 ** -16
    assert dz_err <= (2.0 ** -8 if z.dtype == BF else 0.0) * float(dz_want.norm()) + 2.0 ** -16 * float(dlp.norm())
    return loss, lp, dz


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [None, 30.0])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 64, 1000, 1024, 2048, 2049, 5003])
def test_vocabularies(cuda, V, cap, dtype):
    z, tokens, old, ref, adv = inputs(37, V, dtype, seed=V)
    compare(cuda, z, tokens, old, adv, ref, None, (0.2, 0.28), 0.1, cap)


@pytest.mark.parametrize("N,V", [(1, 1024), (3, 40000), (300, 9000), (9000, 257), (70000, 16), (17000, 2100)])
def test_row_counts(cuda, N, V):
    """Both sides of every choice of waves a row and rows a wave."""
    z, tokens, old, ref, adv = inputs(N, V, BF, seed=N)
    compare(cuda, z, tokens, old, adv, ref, None, (0.2, 0.2), 0.05, 30.0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kl", [0.0, 0.3])
def test_weights_and_rows_that_hold_nothing(cuda, kl, dtype):
    z, tokens, old, ref, adv = inputs(200, 515, dtype, seed=4)
    g = torch.Generator().manual_seed(1)
    w = torch.rand(200, generator=g)
    w[::3] = 0.0
    bad = (z.clone(), old.clone(), ref.clone(), adv.clone())
    for x in bad:
        x[::3] = float("nan")
    bad[0][3] = float("inf")
    tok = tokens.clone()
    tok[::3] = -7
    loss, lp, dz = compare(cuda, bad[0], tok, bad[1], bad[3], bad[2], w, (0.1, 0.3), kl, 30.0, upstream=-2.5)
    assert not bool(lp[::3].any()) and not bool(dz[::3].any())
    # no row at all counts
    import thetascan_amd as ts

    zd = bad[0].to(cuda).requires_grad_()
    loss, lp = ts.policy_loss(zd, tok.to(cuda), old.to(cuda), adv.to(cuda), weights=torch.zeros(200, device=cuda))
    loss.backward()
    assert float(loss) == 0.0 and not bool(zd.grad.any())


def test_clipping_has_the_gradient_of_the_smaller_side(cuda):
    """Both signs of the advantage on both sides of both borders."""
    z = torch.randn(8, 100, generator=torch.Generator().manual_seed(2))
    tokens = torch.arange(8)
    lp = torch.log_softmax(z.double(), -1).gather(-1, tokens[:, None])[:, 0]
    ratio = torch.tensor([0.5, 0.9, 1.1, 1.5, 0.5, 0.9, 1.1, 1.5]).double()
    adv = torch.tensor([1.0, 1, 1, 1, -1, -1, -1, -1])
    _, _, dz = compare(cuda, z, tokens, (lp - ratio.log()).float(), adv, clip=(0.2, 0.3))
    still = [not bool(r.any()) for r in dz]
    assert still == [False, False, False, True, True, False, False, False]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_masked_logits_and_large_ones(cuda, dtype):
    z, tokens, old, ref, adv = inputs(40, 300, dtype, seed=5)
    z[:, ::2] = -float("inf")
    tokens = tokens // 2 * 2 + 1
    z[:, 1] = 80.0
    z[3] = torch.finfo(dtype).min
    old = torch.log_softmax(z.double(), -1).gather(-1, tokens[:, None])[:, 0].float()
    for cap in (None, 30.0):
        import thetascan_amd as ts

        zd = z.to(cuda).requires_grad_()
        loss, lp = ts.policy_loss(zd, tokens.to(cuda), old.to(cuda), adv.to(cuda), softcap=cap)
        zr = z.double().requires_grad_()
        want, lp_want, _ = reference(zr, tokens, old, adv, cap=cap)
        assert float((lp.double().cpu() - lp_want).abs().max()) <= 2.0 ** -17 * 16  # values of up to 16 x 30 log2 e
        (dz,) = torch.autograd.grad(loss, zd)
        assert bool(torch.isfinite(dz).all())


def test_strided_rows_layouts_and_dtypes(cuda):
    import thetascan_amd as ts

    z, tokens, old, ref, adv = inputs(60, 333, BF, seed=6)
    dev = [x.to(cuda) for x in (z, tokens, old, adv, ref)]

    def call(z, tokens, old, adv, ref):
        leaf = z.detach().requires_grad_()
        loss, lp = ts.policy_loss(leaf, tokens, old, adv, ref_log_probs=ref, kl=0.1, softcap=30.0)
        (dz,) = torch.autograd.grad(loss, leaf)
        return loss.detach(), lp, dz

    want = call(*dev)
    wide = torch.zeros(60, 400, dtype=BF, device=cuda)
    for at in (0, 1, 5, 8):
        wide[:, at:at + 333] = dev[0]
        got = call(wide[:, at:at + 333], *dev[1:])
        # (other groupings of a row's sum: rounding apart)
        assert abs(float(got[0]) - float(want[0])) <= 2.0 ** -16
        assert float((got[1] - want[1]).abs().max()) <= 2.0 ** -16
        assert float((got[2].double() - want[2].double()).norm() / want[2].double().norm()) <= 2.0 ** -8
    turned = dev[0].t().contiguous().t()
    for a, b in zip(call(turned, *dev[1:]), want):
        assert torch.equal(a, b)
    shaped = call(dev[0].view(5, 12, 333), *(x.view(5, 12) for x in dev[1:]))
    assert torch.equal(shaped[0], want[0]) and torch.equal(shaped[1].view(-1), want[1])
    assert torch.equal(shaped[2].view(60, 333), want[2])
    assert torch.equal(ts.token_log_probs(dev[0], dev[1], softcap=30.0), want[1])
    empty = ts.policy_loss(dev[0][:0].requires_grad_(), *(x[:0] for x in dev[1:4]))
    assert float(empty[0]) == 0.0 and empty[1].shape == (0,)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [100, 1000, 5000, 70000])
def test_second_backward_and_two_pass_rows(cuda, V, dtype):
    """The gradient of the first backward, of a second one of the same loss with
    another upstream gradient, of rows that take one pass and of rows that take two."""
    import thetascan_amd as ts
    from thetascan_amd import _lib

    z, tokens, old, ref, adv = inputs(21, V, dtype, seed=V)
    want, lp_want, _ = reference(z.double().requires_grad_(), tokens, old, adv, cap=30.0)
    zr = z.double().requires_grad_()
    want, lp_want, _ = reference(zr, tokens, old, adv, cap=30.0)
    dz_want, dlp = torch.autograd.grad(want, (zr, lp_want))
    zd = z.to(cuda).requires_grad_()
    with _lib.record_launches() as recs:
        loss, _ = ts.policy_loss(zd, tokens.to(cuda), old.to(cuda), adv.to(cuda), softcap=30.0)
        first = torch.autograd.grad(loss, zd, retain_graph=True)[0]
        held = first.clone()
        second = torch.autograd.grad(loss, zd, torch.tensor(-3.0, device=cuda), retain_graph=True)[0]
        third = torch.autograd.grad(loss, zd)[0]
    names = [r[0] for r in recs]
    # (21 rows of 70000 are few and long: their scans are split, and loss and gradient take two passes too)
    assert names.count("ts_policy_loss_bwd") == (2 if V == 5000 else 3)
    assert torch.equal(first, held)
    for x, g in ((first, 1.0), (second, -3.0), (third, 1.0)):
        err = float((x.double().cpu() / g - dz_want).norm())
        assert err <= (2.0 ** -8 if dtype == BF else 0.0) * float(dz_want.norm()) + 2.0 ** -16 * float(dlp.norm())
    # an upstream gradient other than one: rounded to bf16 before and after
    loss, _ = ts.policy_loss(zd, tokens.to(cuda), old.to(cuda), adv.to(cuda), softcap=30.0)
    x = torch.autograd.grad(loss * 0.3, zd)[0]
    err = float((x.double().cpu() / 0.3 - dz_want).norm())
    assert err <= (2 * 2.0 ** -8 if dtype == BF else 0.0) * float(dz_want.norm()) + 2.0 ** -15 * float(dlp.norm())


def test_a_token_outside_the_vocabulary_gives_nan(cuda):
    import thetascan_amd as ts

    z, tokens, old, _, adv = (x.to(cuda) for x in inputs(4, 50, F32, seed=7))
    tokens[2] = 50
    loss, lp = ts.policy_loss(z, tokens, old, adv)
    assert torch.isnan(loss) and torch.isnan(lp).tolist() == [False, False, True, False]


def test_graph_replays_and_repeats(cuda):
    import thetascan_amd as ts

    z, tokens, old, ref, adv = (x.to(cuda) for x in inputs(5000, 1024, BF, seed=8))
    z.requires_grad_()

    def step():
        loss, lp = ts.policy_loss(z, tokens, old, adv, ref_log_probs=ref, kl=0.1, softcap=30.0)
        return [loss, lp, *torch.autograd.grad(loss, z)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        with torch.no_grad():
            z.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_compiled_call_is_the_eager_one(cuda):
    import thetascan_amd as ts

    z, tokens, old, _, adv = (x.to(cuda) for x in inputs(30, 100, BF, seed=9))
    z.requires_grad_()

    def f(z):
        return ts.policy_loss(z, tokens, old, adv)[0] * 2.0

    a, b = f(z), torch.compile(f, backend="aot_eager", fullgraph=True)(z)
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, z)[0], torch.autograd.grad(b, z)[0])


def test_a_captured_backward_replayed_more_often_than_its_forward(cuda):
    """Forward and backward in graphs of their own, the backward replayed twice: the
    second gives what the first gave (rows long enough to form loss and gradient in
    one pass, an upstream gradient that is not one)."""
    import thetascan_amd as ts

    z, tokens, old, ref, adv = (x.to(cuda) for x in inputs(5, 2056, BF))

    def loss_of(x):
        return ts.policy_loss(x, tokens, old, adv, ref_log_probs=ref, kl=0.1)[0]

    graphed = torch.cuda.make_graphed_callables(loss_of, (z.clone().requires_grad_(),))
    for seed in (1, 2):
        zr = inputs(5, 2056, BF, seed)[0].to(cuda).requires_grad_()
        loss = graphed(zr)
        got = [torch.autograd.grad(3.0 * loss, zr, retain_graph=True)[0].clone() for _ in range(2)]
        assert torch.equal(got[0], got[1])
        want = torch.autograd.grad(3.0 * loss_of(zr), zr)[0]
        # (one rounding of the row's gradient here, the scaling's second one there)
        assert (got[0].float() - want.float()).abs().max() <= 2 * 2.0 ** -8 * want.float().abs().max()


@pytest.mark.parametrize("V", [64, 2056])
def test_traced_log_probs(cuda, V):
    import thetascan_amd as ts

    z, tokens = (x.to(cuda) for x in inputs(6, V, BF)[:2])
    fn = torch.compile(lambda x, t: ts.token_log_probs(x.view(2, 3, -1), t, softcap=30.0), backend="eager", fullgraph=True)
    got = fn(z, tokens.view(2, 3))
    assert torch.equal(got, ts.token_log_probs(z, tokens, softcap=30.0).view(2, 3)) and not got.requires_grad


def test_traced_loss_of_changing_sizes(cuda):
    import thetascan_amd as ts

    fn = torch.compile(lambda x, t, o, a: ts.policy_loss(x, t, o, a, softcap=30.0), backend="aot_eager", dynamic=True,
                       fullgraph=True)
    for N, V in ((6, 64), (9, 64), (9, 2056)):
        z, tokens, old, _, adv = (x.to(cuda) for x in inputs(N, V, F32))
        z.requires_grad_()
        want, got = ts.policy_loss(z, tokens, old, adv, softcap=30.0), fn(z, tokens, old, adv)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(*(torch.autograd.grad(x[0], z)[0] for x in (want, got)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [77, 2500])
@pytest.mark.parametrize("cap", [0.5, 64.0, 64.5, 1000.0, 1e6, 1e20])
def test_caps_of_any_size(cuda, cap, V, dtype):
    """A cap far above the logits leaves them as they are (to fp32's rounding of logits
    up to 16, 2^-20: within the bars above), one below them binds."""
    z, tokens, old, ref, adv = inputs(9, V, dtype, seed=V)
    y = cap * torch.tanh(z.double() / cap)
    old = (torch.log_softmax(y, -1).gather(-1, tokens[:, None])[:, 0] + 0.4 * (old - ref)).float()
    compare(cuda, z, tokens, old, adv, ref, None, (0.2, 0.28), 0.1, cap)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_few_long_rows(cuda, dtype):
    """Rows whose scans several workgroups share: parts that hold nothing (-inf, the
    type's lowest value), rows of weight zero that hold anything, odd lengths and strides,
    replays of a captured call."""
    import thetascan_amd as ts

    V = 70001
    z, tokens, old, ref, adv = inputs(6, V, dtype, seed=5)
    z[1, :30000] = float("-inf")
    z[2, 9000:] = torch.finfo(dtype).min
    z[3] = float("nan")
    tokens[1], tokens[2], tokens[3] = 40000, 17, -1
    weights = torch.tensor([0.5, 0.25, 0.1, 0.0, 0.3, 0.2])
    old = torch.log_softmax(z.double(), -1).gather(-1, tokens.clamp(0)[:, None])[:, 0].nan_to_num().float() + 0.1 * adv
    compare(cuda, z, tokens, old, adv, ref, weights, (0.2, 0.28), 0.0, None)
    wide = torch.zeros(6, V + 3, dtype=dtype, device=cuda)
    zd = wide[:, 1:V + 1]
    zd.copy_(z)
    lp = ts.token_log_probs(zd[[0, 1, 2, 4, 5]], tokens[[0, 1, 2, 4, 5]].to(cuda))
    args = [x.to(cuda) for x in (tokens, old, adv)]
    w = weights.to(cuda)
    loss, got = ts.policy_loss(zd, *args, weights=w)
    assert torch.equal(got[[0, 1, 2, 4, 5]], lp) and got[3] == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ts.policy_loss(zd, *args, weights=w)
    for _ in range(3):
        zd[0].add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        again = ts.policy_loss(zd, *args, weights=w)
        assert torch.equal(held[0], again[0]) and torch.equal(held[1], again[1])
