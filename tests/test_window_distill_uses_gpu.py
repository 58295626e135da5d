"""Windowed attention, distillation and generation in the uses that their documents allow: saved tensors
offloaded or formed again, a backward captured without its forward, autocast, scales at the ends of fp32, settings that are
no numbers."""
from __future__ import annotations

import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tests.test_distill_gpu import teacher
from tests.test_generation_gpu import _model
from tests.test_window_gpu import inputs, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 20])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_offloaded_and_checkpointed(cuda, d, dtype):
    import thetascan_amd as ts

    q, k, v, do = (x.to(cuda) for x in inputs(2, 4, 2, 150, d, dtype))
    lengths = torch.tensor([150, 77], device=cuda)

    def f(q, k, v):
        return ts.windowed_attention(q, k, v, window=40, sinks=2, lengths=lengths)

    def grads(g, **kw):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = g(*leaves, **kw)
        return [out, *torch.autograd.grad(out, leaves, do)]

    base = grads(f)
    again = grads(lambda *x: checkpoint(f, *x, use_reentrant=False))
    with torch.autograd.graph.save_on_cpu():
        offloaded = grads(f)
    for got in (again, offloaded):
        assert all(torch.equal(a, b) for a, b in zip(base, got))


@pytest.mark.parametrize("V", [1000, 5001])
def test_distillation_offloaded_and_checkpointed(cuda, V):
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(V)
    z = (2.0 * torch.randn(33, V, generator=g)).bfloat16()
    ids, lps = (x.to(cuda) for x in teacher(z, 12, g))
    z = z.to(cuda)

    def f(z):
        return ts.distill_loss(z, ids, lps, temperature=1.3, softcap=30.0)[0]

    def grads(h, scale):
        leaf = z.detach().requires_grad_(True)
        loss = h(leaf) * scale
        return [loss, *torch.autograd.grad(loss, [leaf])]

    for scale in (1.0, 3.0):
        base = grads(f, scale)
        again = grads(lambda z: checkpoint(f, z, use_reentrant=False), scale)
        with torch.autograd.graph.save_on_cpu():
            offloaded = grads(f, scale)
        for got in (again, offloaded):
            assert all(torch.equal(a, b) for a, b in zip(base, got))


@pytest.mark.parametrize("V", [1000, 5001])
def test_a_distillation_backward_captured_alone(cuda, V):
    """The forward runs before the capture; every replay takes the upstream gradient of its time."""
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(V)
    z = (2.0 * torch.randn(33, V, generator=g)).bfloat16()
    ids, lps = (x.to(cuda) for x in teacher(z, 12, g))
    up = torch.ones((), device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = z.to(cuda).requires_grad_(True)
        torch.autograd.grad(ts.distill_loss(warm, ids, lps)[0], warm, up)
        leaf = z.to(cuda).requires_grad_(True)
        loss = ts.distill_loss(leaf, ids, lps)[0]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            (held,) = torch.autograd.grad(loss, leaf, up)
    torch.cuda.current_stream().wait_stream(side)
    for x in (2.0, 1.0, -0.5, 1.0):
        up.fill_(x)
        graph.replay()
        torch.cuda.synchronize()
        other = z.to(cuda).requires_grad_(True)
        (want,) = torch.autograd.grad(ts.distill_loss(other, ids, lps)[0], other, torch.tensor(x, device=cuda))
        # (a unit gradient stands from the forward, another is formed by the backward: one rounding apart)
        assert torch.allclose(held.float(), want.float(), rtol=2.0 ** -7, atol=1e-30)


@pytest.mark.parametrize("memory", ["theta", "delta"])
def test_generation_under_autocast(cuda, memory):
    """An fp32 model under autocast to bf16 generates as it trains: its products in bf16."""
    model = _model(memory, torch.float32, cuda, window=16, sinks=2)
    g = torch.Generator().manual_seed(1)
    idx = torch.randint(0, 1024, (3, 21), generator=g).to(cuda)
    u = torch.rand(3, 25, generator=g).to(cuda)
    with torch.autocast("cuda", torch.bfloat16):
        tokens, lps = model.generate(idx, u, top_k=50)
        whole = torch.cat([idx, tokens], 1)
        want = model.log_probs(whole[:, :-1], whole[:, 1:])[:, 20:]
    # (bf16 logits of some ones: a rounding or two of 2^-8 at each of nine layers' ends)
    assert torch.isfinite(lps).all() and (lps - want).abs().max() < 0.15


@pytest.mark.parametrize("scale", [1.2e-38, 1e-30, 2e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_at_the_ends_of_fp32(cuda, scale, dtype):
    """Scores of next to zero: every query's mean of the values that it sees; the largest scale that is
    taken: of scores far apart, the highest alone."""
    import thetascan_amd as ts

    T = 100
    q, k, v, do = (x.to(cuda) for x in inputs(1, 2, 2, T, 64, dtype))
    seen = visible(T, 30, 2)
    if scale > 1.0:
        q, k = (torch.zeros_like(x) for x in (q, k))
        k[..., 0] = torch.arange(T, device=cuda).remainder(30).to(dtype)  # (within a window, the highest is one token)
        q[..., 0] = 1e-36
        seen = visible(T, 30, 0)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    sinks = 2 if scale < 1.0 else 0
    out = ts.windowed_attention(*leaves, window=30, sinks=sinks, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    if scale < 1.0:
        P = seen.double() / seen.double().sum(-1, keepdim=True)
    else:
        s = torch.where(seen, k[0, 0, :, 0].double().cpu(), -math.inf)
        P = torch.nn.functional.one_hot(s.argmax(-1), T).double()
    want = (P @ v.double().cpu(), P.T @ do.double().cpu())
    for x, y in zip((out, grads[2]), want):
        assert torch.allclose(x.detach().double().cpu(), y, rtol=2.0 ** -7, atol=2.0 ** -7 if dtype == torch.bfloat16 else 1e-5)
    assert all(torch.isfinite(x).all() for x in grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_cache_filled_from_itself(cuda, dtype):
    """Tokens dropped from the front: the slots' rows move within the cache, each read before it is written."""
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(3)
    for drop, sinks in ((1, 0), (3, 2), (500, 16)):
        caches = [torch.randn(3, 4, 2000, 64, generator=g).to(dtype).to(cuda) for _ in range(2)]
        want = [x.clone() for x in caches]
        rows = [x[:, :, drop:] for x in caches]
        for x in want:
            x[:, :, :2000 - drop] = x[:, :, drop:].clone()
        ts.fill_window_cache(*rows, *caches, sinks=sinks)
        assert all(torch.equal(x, y) for x, y in zip(caches, want))


@pytest.mark.parametrize("V", [100, 9000])
def test_a_row_of_a_setting_that_is_no_number_draws_nothing(cuda, V):
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(4)
    z, u = torch.randn(4, V, generator=g).to(cuda), torch.rand(4, generator=g).to(cuda)
    usual = dict(temperature=torch.full((4,), 0.8), top_p=torch.full((4,), 0.9), min_p=torch.full((4,), 0.01))
    want = ts.sample_tokens(z, u, **{n: x.to(cuda) for n, x in usual.items()})
    for row, name in enumerate(usual):
        one = {n: x.clone() for n, x in usual.items()}
        one[name][row] = math.nan
        for more in (dict(), dict(top_k=7)):
            tokens, lps = ts.sample_tokens(z, u, **{n: x.to(cuda) for n, x in one.items()}, **more)
            assert int(tokens[row]) == -1 and math.isnan(float(lps[row]))
            if not more:
                others = torch.arange(4, device=cuda) != row
                assert torch.equal(tokens[others], want[0][others]) and torch.equal(lps[others], want[1][others])
