"""Windowed attention at the sizes of training batches, whose kernels own more rows than those of
small calls: 32 queries a wave from 256 workgroups on, 128 keys a workgroup (bf16, heads of at most
64), and workgroups that walk the query heads of a key head one after the other (from 128 on); sinks
over several stretches of queries, padded batches, strides, values that are not finite.  Against
float64 by the bars of tests/test_window_gpu.py, on some of the sequences.
"""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_window_gpu import U, close, inputs, reference, run, visible

pytestmark = pytest.mark.gpu

# 64 and 128 keys a workgroup, two and four query heads one after the other, one to five stretches of sinks' queries
SHAPES = [(8, 8, 4, 577, 64), (16, 8, 4, 391, 64), (16, 16, 4, 385, 64), (4, 16, 8, 1100, 64), (8, 8, 2, 577, 128),
          (2, 16, 8, 1290, 128), (16, 8, 4, 391, 40), (8, 8, 2, 577, 80), (4, 16, 8, 1100, 8)]


def on_some(B, T, q, k, v, do, lengths=None):
    """The sequences that are compared: few, where they are long."""
    some = list(range(0, B, 5 if T < 600 else B))
    return some, [x[some] for x in (q, k, v, do)], None if lengths is None else lengths[some]


@pytest.mark.parametrize("B,H,Hk,T,d", SHAPES)
@pytest.mark.parametrize("window,sinks", [(100, 0), (200, 4), (33, 130), (64, 64), (None, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_workgroups(cuda, B, H, Hk, T, d, window, sinks, dtype):
    q, k, v, do = inputs(B, H, Hk, T, d, dtype, T + d)
    some, few, _ = on_some(B, T, q, k, v, do)
    want, bars = reference(*few, window, sinks)
    for name, x, y, bar in zip(("out", "dq", "dk", "dv"), run(cuda, q, k, v, do, window=window, sinks=sinks), want, bars):
        close(name, x[some], y, bar)


@pytest.mark.parametrize("B,H,Hk,T,d", [(8, 8, 4, 577, 64), (16, 8, 4, 391, 64), (8, 8, 2, 577, 128), (8, 8, 2, 577, 80)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_batches(cuda, B, H, Hk, T, d, dtype):
    """Rows past a length are not read (they hold NaN), and give zeros."""
    lengths = torch.tensor([T, 0, 1, 130, T - 1, 64, 300, 257] * 2)[:B]
    q, k, v, do = inputs(B, H, Hk, T, d, dtype)
    past = (torch.arange(T) >= lengths[:, None])[:, None, :, None]
    bad = [x.masked_fill(past, math.nan) for x in (q, k, v, do)]
    for window, sinks in ((90, 7), (33, 130)):
        got = run(cuda, *bad, window=window, sinks=sinks, lengths=lengths.to(cuda))
        want, bars = reference(*(x[:8] for x in (q, k, v, do)), window, sinks, lengths[:8])
        for name, x, y, bar in zip(("out", "dq", "dk", "dv"), got, want, bars):
            close(name, x[:8], y, bar)
            assert not x.detach().masked_select(past.to(cuda).expand_as(x)).any()


@pytest.mark.parametrize("B,H,Hk,T,d", [(8, 8, 4, 577, 64), (16, 8, 4, 391, 64), (8, 8, 2, 577, 128)])
def test_strides(cuda, B, H, Hk, T, d):
    """Heads before tokens, rows of a wider matrix, every second token and unaligned rows give the same
    as token-major inputs, bit for bit."""
    import thetascan_amd as ts

    q, k, v, do = (x.to(cuda) for x in inputs(B, H, Hk, T, d, torch.bfloat16))

    def unaligned(x):
        return torch.empty(x.numel() + 1, dtype=x.dtype, device=cuda)[1:].view(x.shape).copy_(x)

    base = None
    for f in (lambda x: x, lambda x: x.contiguous(), lambda x: torch.cat([x, x, x], -1)[..., d:2 * d],
              lambda x: torch.stack([x, x], 3).flatten(2, 3)[:, :, ::2], unaligned):
        leaves = [f(x).detach().requires_grad_(True) for x in (q, k, v)]
        out = ts.windowed_attention(*leaves, window=70, sinks=9)
        got = [out, *torch.autograd.grad(out, leaves, f(do))]
        base = got if base is None else base
        for x, y in zip(got, base):
            assert torch.equal(x, y)


@pytest.mark.parametrize("B,H,Hk,T,d", [(8, 8, 4, 577, 64), (8, 8, 2, 577, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_reaches_who_sees_it_alone(cuda, B, H, Hk, T, d, bad):
    import thetascan_amd as ts

    window, sinks, dtype = 40, 3, torch.bfloat16
    q, k, v, _ = (x.to(cuda) for x in inputs(B, H, Hk, T, d, dtype))
    seen = visible(T, window, sinks).to(cuda)
    clean = ts.windowed_attention(q, k, v, window=window, sinks=sinks)
    rep = H // Hk
    for at in (0, 70, 300, T - 1):
        for name in "kvq":
            x = {"q": q.clone(), "k": k.clone(), "v": v.clone()}
            x[name][0, 1, at, 5] = bad
            out = ts.windowed_attention(*(x[n] for n in "qkv"), window=window, sinks=sinks)
            heads = range(rep, 2 * rep) if name != "q" else [1]
            others = [h for h in range(H) if h not in heads]
            assert torch.equal(out[1:], clean[1:]) and torch.equal(out[0, others], clean[0, others])
            free = ~seen[:, at] if name != "q" else torch.arange(T, device=cuda) != at
            for h in heads:
                # (the workgroups that go over their tiles again add in another order)
                assert torch.allclose(out[0, h][free], clean[0, h][free], rtol=2 * U[dtype] + 1e-5, atol=2e-2)
                if name == "v":
                    assert torch.equal(~torch.isfinite(out[0, h, :, 5]), seen[:, at])


@pytest.mark.parametrize("B,H,Hk,T,d,sinks", [(16, 8, 8, 1300, 64, 1100), (16, 16, 8, 1300, 16, 700), (4, 8, 8, 1300, 128, 1200),
                                              (1, 8, 2, 2100, 64, 1500)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_sinks(cuda, B, H, Hk, T, d, sinks, dtype):
    """So many of them that their queries are not cut into stretches, or into few."""
    q, k, v, do = inputs(B, H, Hk, T, d, dtype, T + d)
    want, bars = reference(*(x[-1:] for x in (q, k, v, do)), 20, sinks)
    for name, x, y, bar in zip(("out", "dq", "dk", "dv"), run(cuda, q, k, v, do, window=20, sinks=sinks), want, bars):
        close(name, x[-1:], y, bar)
