"""distill_loss (ts_distill_fwd, ts_distill_bwd) against float64.

fp32 sums of exponentials: terms off by (|x - max| + 8) 2^-22 of themselves at most (the
logit's, the cap's and the difference's rounding, and the exponential's), and a sum of V
terms by lanes; the K terms and the rows are fp64.  With q the student's shares, that is
d = sum q (|x| + |x - max| + 8) 2^-22 + (V / 64 + 32) 2^-24 for the log of the sum, and
of the others' share alike.  A row's loss: M d + 2^-24 of itself; its gradient:
w / temperature (q (M + P_r / Q_r) (d + its own term's error) + P 2^-22) and its rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def reference(z, ids, lps, weights, temperature, tail, cap):
    """(loss, each, dz) and their bars in float64, by the definition."""
    u, (N, V) = U[z.dtype], z.shape
    w = torch.full((N,), 1.0 / N, dtype=torch.float64) if weights is None else weights.double()
    used = (w != 0)[:, None]
    z = torch.where(used, z.double(), 0.0)
    y = cap * torch.tanh(z / cap) if cap else z
    slope = (1.0 / torch.cosh(z / cap) ** 2 if cap else torch.ones_like(z)) / temperature
    x = y / temperature
    lq = torch.log_softmax(x, -1)
    q = lq.exp()
    there = ids >= 0
    at = ids.clamp(min=0)
    P = torch.where(there, lps.double().exp(), 0.0)
    if not tail:
        P = P / P.sum(-1, keepdim=True)
    teacher = torch.zeros(N, V, dtype=torch.float64).scatter_add_(-1, at, P)
    member = torch.zeros(N, V).scatter_add_(-1, at, there.float()) > 0
    each = torch.special.xlogy(teacher, teacher).sum(-1) - torch.where(teacher > 0, teacher * lq, 0.0).sum(-1)
    rest = torch.where(member, 0.0, q)
    Q = rest.sum(-1)
    M = teacher.sum(-1)
    left = torch.zeros(N, dtype=torch.float64)
    if tail:
        left = torch.where(Q > 0, (1.0 - M).clamp(min=0.0), 0.0)
        each = each + torch.where(left > 0, left * (left.log() - Q.log()), 0.0)
        M = M + left
    ratio = torch.where(left > 0, left / Q, 0.0)[:, None]
    grad = q * M[:, None] - teacher - rest * ratio
    dz = w[:, None] * grad * slope
    own = (x.abs() + lq.abs() + (x - x.amax(-1, keepdim=True)).abs() + 8.0) * 2.0 ** -22
    sums = (V / 64 + 32) * 2.0 ** -24
    d = (q * own).sum(-1) + sums
    dr = torch.where(Q > 0, (rest * own).sum(-1) / Q, 0.0) + sums
    each_bar = M * d + left * dr + 2.0 ** -24 * each.abs() + (P * lps.abs().masked_fill(~there, 0.0)).sum(-1) * 2.0 ** -40
    each = torch.where(used[:, 0], each, 0.0)
    dz_bar = u * dz.abs() + w.abs()[:, None] * slope * (q * (M[:, None] + ratio) * (d[:, None] + dr[:, None] + own)
                                                        + teacher * 2.0 ** -22) + 2.0 ** -22 * dz.abs() + 1e-38
    if cap:  # (the slope's own rounding)
        dz_bar = dz_bar + w.abs()[:, None] * grad.abs() * 2.0 ** -21 / temperature
    loss = (w * each).sum()
    return (loss, each, dz), ((w.abs() * each_bar).sum() + 2.0 ** -24 * loss.abs(), each_bar, dz_bar)


def run(cuda, z, ids, lps, weights=None, g=None, **kw):
    import thetascan_amd as ts

    leaf = z.to(cuda).requires_grad_(True)
    loss, each = ts.distill_loss(leaf, ids.to(cuda), lps.to(cuda), weights=None if weights is None else weights.to(cuda), **kw)
    (dz,) = torch.autograd.grad(loss, leaf, None if g is None else g.to(cuda))
    torch.cuda.synchronize()
    return loss.detach().cpu(), each.cpu(), dz.cpu()


def teacher(z, K, g, temperature=1.0, spread=0.5):
    y = z.float().nan_to_num(0.0) + spread * torch.randn(z.shape, generator=g)
    lp, ids = torch.log_softmax(y / temperature, -1).topk(K, -1)
    order = torch.rand(lp.shape, generator=g).argsort(-1)
    return ids.gather(-1, order), lp.gather(-1, order)


def close(got, want, bars):
    for name, x, y, bar in zip(("loss", "each", "dz"), got, want, bars):
        err = (x.double() - y).abs()
        worst = float((err / bar.clamp(min=1e-45)).max()) if err.numel() else 0.0
        print(f"{name}: {worst:.3f} of its bar", flush=True)
        assert worst <= 1.0, name


@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (3, 2, 1), (5, 64, 64), (7, 1000, 20), (64, 1024, 32), (9, 2048, 100),
                                   (9, 2049, 100), (6, 5003, 256), (3, 32768, 64), (2, 131072, 300), (2, 300001, 8)])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sizes(cuda, N, V, K, tail, dtype):
    g = torch.Generator().manual_seed(V + K)
    z = (2.5 * torch.randn(N, V, generator=g)).to(dtype)
    ids, lps = teacher(z, K, g)
    close(run(cuda, z, ids, lps, tail=tail), *reference(z, ids, lps, None, 1.0, tail, None))


@pytest.mark.parametrize("cap,temperature", [(None, 2.0), (30.0, 1.0), (5.0, 0.5), (1e4, 3.0)])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V", [777, 4099])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_caps_and_temperatures(cuda, cap, temperature, tail, V, dtype):
    g = torch.Generator().manual_seed(V)
    z = (6.0 * torch.randn(11, V, generator=g)).to(dtype)
    ids, lps = teacher(z, 17, g, temperature)
    close(run(cuda, z, ids, lps, tail=tail, softcap=cap, temperature=temperature),
          *reference(z, ids, lps, None, temperature, tail, cap))


@pytest.mark.parametrize("V", [600, 3001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_missing_tokens_and_agreement(cuda, V, dtype):
    """Rows of weight zero hold anything; ids below zero are no tokens (down to none of a row); where
    teacher and student agree, the loss is its digits (the shares of all others of 1e-6)."""
    g = torch.Generator().manual_seed(V)
    N, K = 12, 10
    z = 3.0 * torch.randn(N, V, generator=g)
    z[4:8, :6] += 16.0
    z = z.to(dtype)
    ids, lps = teacher(z, K, g, spread=0.1)
    ids[2, 3:], ids[3] = -1, -7
    lps[2, 5] = math.nan
    weights = torch.rand(N, generator=g)
    weights[[0, 9]] = 0.0
    weights[10] = -0.5
    want = reference(z, ids, lps.nan_to_num(0.0), weights, 1.0, True, None)
    z[0], ids[9], lps[9] = math.nan, V + 5, math.inf
    got = run(cuda, z, ids, lps, weights)
    close(got, *want)
    assert not got[2][[0, 9]].any() and not got[1][[0, 9]].any()


def test_wrong_tokens_are_nan(cuda):
    g = torch.Generator().manual_seed(1)
    for V in (500, 5000):
        z = torch.randn(4, V, generator=g)
        ids, lps = teacher(z, 5, g)
        ids[1, 2] = ids[1, 4]
        ids[2, 0] = V
        loss, each, dz = run(cuda, z, ids, lps)
        bad = torch.tensor([False, True, True, False])
        assert math.isnan(float(loss)) and torch.equal(torch.isnan(each), bad)
        assert torch.isnan(dz[bad]).all() and torch.isfinite(dz[~bad]).all()


def test_forbidden_tokens(cuda):
    """-inf logits outside the teacher's tokens: shares and gradients of zero; all others forbidden:
    no tail; a teacher's token forbidden: an infinite loss."""
    g = torch.Generator().manual_seed(2)
    for V in (300, 3000):
        z = torch.randn(3, V, generator=g)
        ids, lps = teacher(z, 4, g)
        z[0, (torch.arange(V) % 7 == 0) & ~torch.isin(torch.arange(V), ids[0])] = -math.inf
        z[1, ~torch.isin(torch.arange(V), ids[1])] = -math.inf
        z[2, ids[2, 0]] = -math.inf
        loss, each, dz = run(cuda, z, ids, lps)
        q = torch.softmax(z[0].double(), -1)
        P = lps[0].double().exp()
        Q = 1.0 - q[ids[0]].sum()
        want = (P * (lps[0].double() - q[ids[0]].log())).sum() + (1 - P.sum()) * ((1 - P.sum()).log() - Q.log())
        assert abs(float(each[0]) - float(want)) < 1e-5 * abs(float(want)) + 1e-6
        assert not dz[0][z[0] == -math.inf].any() and torch.isfinite(dz[:2]).all()
        lq = torch.log_softmax(z[1, ids[1]].double(), -1)
        P = lps[1].double().exp()
        assert abs(float(each[1]) - float((P * (lps[1].double() - lq)).sum())) < 1e-6
        assert float(each[2]) == math.inf


def test_upstream_gradients_strides_and_shapes(cuda):
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(3)
    z = torch.randn(6, 999, generator=g).bfloat16()
    ids, lps = teacher(z, 8, g)
    base = run(cuda, z, ids, lps)
    for scale in (3.0, 0.0, -0.5):
        got = run(cuda, z, ids, lps, g=torch.tensor(scale))
        assert torch.equal(got[0], base[0])
        assert torch.allclose(got[2].double(), base[2].double() * scale, rtol=2.0 ** -7, atol=1e-30)
    wide = torch.randn(6, 1007).bfloat16()
    wide[:, 3:1002] = z
    leaf = wide.to(cuda)[:, 3:1002].unflatten(0, (2, 3)).detach().requires_grad_(True)
    loss, each = ts.distill_loss(leaf, ids.to(cuda).view(2, 3, 8), lps.to(cuda).view(2, 3, 8))
    loss.backward()
    assert each.shape == (2, 3)
    # (unaligned rows are spread over the lanes in another way: the same bars, not the same bits)
    close((loss.detach().cpu(), each.flatten().cpu(), leaf.grad.flatten(0, 1).cpu()), *reference(z, ids, lps, None, 1.0, True, None))
    loss, each = ts.distill_loss(torch.zeros(0, 50, device=cuda, requires_grad=True), ids[:0].to(cuda), lps[:0].to(cuda))
    loss.backward()
    assert float(loss) == 0.0 and each.shape == (0,)


def test_gradients_against_differences(cuda):
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(4)
    for V in (200, 2500):
        z = torch.randn(5, V, generator=g).to(cuda)
        ids, lps = (x.to(cuda) for x in teacher(z.cpu(), 6, g))
        way = torch.randn(5, V, generator=g).to(cuda)
        leaf = z.clone().requires_grad_(True)
        kw = dict(temperature=1.5, softcap=8.0)
        (dz,) = torch.autograd.grad(ts.distill_loss(leaf, ids, lps, **kw)[0], leaf)
        slope = float((dz.double() * way.double()).sum())
        h = 2.0 ** -6
        up, down = (ts.distill_loss(z + c * way, ids, lps, **kw)[1].double().mean() for c in (h, -h))
        # (third derivatives of some ones over h^2 / 6, and fp32 losses of some ones over 2 h)
        assert abs(float(up - down) / (2 * h) - slope) < 3e-4


def test_compiled_and_captured(cuda):
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(5)
    for V in (1024, 6001):
        data = [(2.0 * torch.randn(33, V, generator=g)).bfloat16().to(cuda) for _ in range(3)]
        ids, lps = (x.to(cuda) for x in teacher(data[0].cpu(), 12, g))

        def f(z):
            return ts.distill_loss(z, ids, lps, temperature=1.3, softcap=30.0)

        leaf = data[0].clone().requires_grad_(True)

        def step():
            loss, each = f(leaf)
            return [loss, each, *torch.autograd.grad(loss, leaf)]

        base = step()
        loss, each = torch.compile(f, fullgraph=True)(leaf)
        got = [loss, each, *torch.autograd.grad(loss, leaf)]
        assert all(torch.equal(a, b) for a, b in zip(base, got))
        with torch.no_grad():
            assert torch.equal(f(leaf)[0], base[0].detach())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        del base, got, loss, each
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for z in (data[1], data[2], data[0]):
            with torch.no_grad():
                leaf.copy_(z)
            want = [x.detach().clone() for x in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a.detach(), b) for a, b in zip(held, want))
        (g1,) = torch.autograd.grad(f(leaf)[0], leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g1.float().sum().backward()
