"""Windowed attention with sinks (ts_window_attention_fwd, ts_window_attention_bwd)
against float64, and its refusals' counterparts: padded batches, strides, values that are
not finite, graphs.

Every element has a bar of its own, from the roundings on its way (u: bf16 2^-8, fp32 2^-24;
e: fp32 scores of d products, their exponential and a sum of T terms):

* out:   u |out| + (u + e) sum_j P |v|                          (P enters its product rounded)
* dv:    u |dv| + (u + e) sum_i P |dout|
* dS:    E = (u + e) |dS| + P (what D and dP are off by); D is a product with the rounded out
* dq:    u |dq| + scale sum_j E |k|, and dk the same over the queries
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def visible(T, window, sinks):
    i, j = torch.arange(T)[:, None], torch.arange(T)
    return (j <= i) & ((i - j < window) | (j < sinks))


def reference(q, k, v, dout, window, sinks, lengths=None, scale=None):
    """(values, bars) of out, dq, dk, dv in float64, from the formulas."""
    u = U[q.dtype]
    B, H, T, d = q.shape
    Hk, rep = k.shape[1], H // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    seen = visible(T, T if window is None else window, sinks).expand(B, 1, T, T)
    on = torch.ones(B, 1, T, 1, dtype=torch.bool)
    if lengths is not None:
        on = (torch.arange(T) < lengths[:, None])[:, None, :, None]
        seen = seen & on & on.transpose(2, 3)
    q, k, v, dout = (torch.where(on, x.double(), 0.0) for x in (q, k, v, dout))
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = scale * (q @ k.transpose(2, 3))
    e = 2 * (d + 16) * 2.0 ** -24 * float((scale * (q.abs() @ k.abs().transpose(2, 3))).max()) + (T + 64) * 2.0 ** -23
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    P = (s - torch.where(top > -math.inf, top, 0.0)).exp()
    P = P / P.sum(-1, keepdim=True).clamp(min=1e-300)
    out = P @ v
    out_bar = u * out.abs() + (u + e) * (P @ v.abs())
    dP = dout @ v.transpose(2, 3)
    dP_bar = d * 2.0 ** -24 * (dout.abs() @ v.abs().transpose(2, 3))
    D = (dout * out).sum(-1, keepdim=True)
    D_bar = (dout.abs() * (out_bar + d * 2.0 ** -24 * out.abs())).sum(-1, keepdim=True)
    dS = P * (dP - D)
    E = (u + e) * dS.abs() + P * (dP_bar + D_bar)

    def shared(x):
        return x.reshape(B, Hk, rep, T, d).sum(2)

    dq, dk, dv = scale * (dS @ k), scale * shared(dS.transpose(2, 3) @ q), shared(P.transpose(2, 3) @ dout)
    tiny = 1e-30
    bars = [out_bar + tiny, u * dq.abs() + scale * ((E + T * 2.0 ** -24 * dS.abs()) @ k.abs()) + tiny,
            u * dk.abs() + scale * shared((E + rep * T * 2.0 ** -24 * dS.abs()).transpose(2, 3) @ q.abs()) + tiny,
            u * dv.abs() + (u + e + rep * T * 2.0 ** -24) * shared(P.transpose(2, 3) @ dout.abs()) + tiny]
    return [out, dq, dk, dv], bars


def inputs(B, H, Hk, T, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(B, T, H, d, generator=g) for _ in range(2))
    k, v = (torch.randn(B, T, Hk, d, generator=g) for _ in range(2))
    return [(x * c).to(dtype).transpose(1, 2) for x, c in ((q, 1.5), (k, 1.0), (v, 1.0), (do, 1.0))]


def close(name, got, want, bar):
    err = (got.detach().double().cpu() - want).abs()
    worst = float((err / bar).max()) if err.numel() else 0.0
    print(f"{name}: {worst:.3f} of its bar", flush=True)
    assert got.shape == want.shape and worst <= 1.0, name


def run(cuda, q, k, v, dout, **kw):
    import thetascan_amd as ts

    leaves = [x.to(cuda).requires_grad_(True) for x in (q, k, v)]
    out = ts.windowed_attention(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, dout.to(cuda))
    torch.cuda.synchronize()
    return [out, *grads]


@pytest.mark.parametrize("T,window,sinks", [
    (1, 1, 0), (1, 5, 3), (2, 1, 1), (63, 64, 0), (64, 1, 0), (65, 64, 1), (129, 2, 128), (130, 33, 3), (200, 1, 2),
    (257, 64, 65), (300, 100, 4), (300, None, 0), (300, 299, 1), (321, 17, 200), (448, 63, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows_and_sinks(cuda, T, window, sinks, dtype):
    q, k, v, do = inputs(2, 4, 2, T, 64, dtype, T)
    want, bars = reference(q, k, v, do, window, sinks)
    for name, *x in zip(("out", "dq", "dk", "dv"), run(cuda, q, k, v, do, window=window, sinks=sinks), want, bars):
        close(name, *x)


@pytest.mark.parametrize("B,H,Hk,T,d", [(1, 4, 2, 700, 64), (1, 4, 2, 700, 128), (4, 2, 2, 1200, 64), (4, 2, 2, 1200, 128),
                                        (1, 1, 1, 1400, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sinks_of_many_queries(cuda, B, H, Hk, T, d, dtype):
    """Sinks whose queries take several stretches, with the query heads apart and together."""
    q, k, v, do = inputs(B, H, Hk, T, d, dtype, T)
    want, bars = reference(q, k, v, do, 20, 70)
    for name, *x in zip(("out", "dq", "dk", "dv"), run(cuda, q, k, v, do, window=20, sinks=70), want, bars):
        close(name, *x)


@pytest.mark.parametrize("H,Hk,d", [(1, 1, 128), (6, 2, 128), (8, 1, 80), (3, 3, 16), (4, 4, 40), (2, 1, 20), (2, 2, 1),
                                    (4, 2, 96), (5, 5, 65)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_heads_and_widths(cuda, H, Hk, d, dtype):
    q, k, v, do = inputs(2, H, Hk, 150, d, dtype, d)
    want, bars = reference(q, k, v, do, 70, 5)
    for name, *x in zip(("out", "dq", "dk", "dv"), run(cuda, q, k, v, do, window=70, sinks=5), want, bars):
        close(name, *x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_batch(cuda, dtype):
    """Rows past a length are not read (they hold NaN), and give zeros."""
    T = 200
    lengths = torch.tensor([0, 1, 64, 137, 200])
    q, k, v, do = inputs(5, 4, 2, T, 64, dtype)
    want, bars = reference(q, k, v, do, 50, 7, lengths)
    past = (torch.arange(T) >= lengths[:, None])[:, None, :, None]
    bad = [x.masked_fill(past, math.nan) for x in (q, k, v, do)]
    for kind in (torch.int64, torch.int32):
        got = run(cuda, *bad, window=50, sinks=7, lengths=lengths.to(cuda, kind))
        for name, x, y, bar in zip(("out", "dq", "dk", "dv"), got, want, bars):
            close(name, x, y, bar)
            assert not x.detach().masked_select(past.to(cuda).expand_as(x)).any()
    # lengths outside [0, T] are clamped
    got = run(cuda, q, k, v, do, window=50, sinks=7, lengths=torch.tensor([-3, 1, 64, 137, 999], device=cuda))
    for name, x, y, bar in zip(("out", "dq", "dk", "dv"), got, want, bars):
        close(name, x, y, bar)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_any_strides(cuda, dtype):
    """Heads before tokens, rows of a wider matrix, every second token, unaligned rows and broadcast
    ones give the same as contiguous inputs, bit for bit."""
    import thetascan_amd as ts

    q, k, v, do = (x.to(cuda) for x in inputs(2, 4, 2, 100, 64, dtype))

    def tokens_of(x, f):
        leaf = f(x).requires_grad_(True)
        return leaf

    def contiguous(x):
        return x.contiguous()

    def wider(x):
        return torch.cat([x, x, x], -1)[..., 64:128]

    def seconds(x):
        return torch.stack([x, x], 3).flatten(2, 3)[:, :, ::2]

    def unaligned(x):
        flat = torch.empty(x.numel() + 1, dtype=dtype, device=cuda)
        return flat[1:].view(x.shape).copy_(x)

    base = None
    for f in (contiguous, lambda x: x, wider, seconds, unaligned):
        leaves = [f(x).detach().requires_grad_(True) for x in (q, k, v)]
        out = ts.windowed_attention(*leaves, window=30, sinks=3)
        got = [out, *torch.autograd.grad(out, leaves, f(do))]
        base = got if base is None else base
        for x, y in zip(got, base):
            assert torch.equal(x, y)
    one = v[:, :, :1].detach().requires_grad_(True)
    out = ts.windowed_attention(q, k, one.expand(-1, -1, 100, -1), window=30, sinks=3)
    (g,) = torch.autograd.grad(out, one, torch.ones((), dtype=dtype, device=cuda).expand_as(out))
    assert torch.allclose(out.float(), one.float().repeat_interleave(2, 1).expand_as(out), rtol=2.0 ** -6, atol=0)
    # (every query's shares add to one: 100 queries of two heads on each key head)
    assert torch.allclose(g.float(), torch.full_like(g, 200.0).float(), rtol=2.0 ** -6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_reaches_who_sees_it_alone(cuda, dtype, bad):
    import thetascan_amd as ts

    T, window, sinks = 200, 20, 3
    q, k, v, _ = inputs(1, 2, 2, T, 64, dtype)
    seen = visible(T, window, sinks)
    clean = ts.windowed_attention(q.to(cuda), k.to(cuda), v.to(cuda), window=window, sinks=sinks)
    for at in (0, 40, 70, 199):
        for name in ("k", "v", "q"):
            x = {"q": q.clone(), "k": k.clone(), "v": v.clone()}
            x[name][0, 1, at, 5] = bad
            out = ts.windowed_attention(*(x[n].to(cuda) for n in "qkv"), window=window, sinks=sinks)
            assert torch.equal(out[0, 0], clean[0, 0])
            free = ~seen[:, at] if name != "q" else torch.arange(T) != at
            # (the workgroups that go over their tiles again add in another order)
            assert torch.allclose(out[0, 1][free.to(cuda)], clean[0, 1][free.to(cuda)], rtol=2 * U[dtype] + 1e-5, atol=2e-2 if dtype == torch.bfloat16 else 1e-5)
            if name == "v":
                hit = ~torch.isfinite(out[0, 1, :, 5]).cpu()
                assert torch.equal(hit, seen[:, at])
                assert torch.isfinite(out[0, 1][:, torch.arange(64) != 5]).all()


def test_gradients_against_differences(cuda):
    """fp32: the directional derivative of a random functional, central differences of h = 2^-7."""
    import thetascan_amd as ts

    q, k, v, do = (x.to(cuda) for x in inputs(1, 2, 1, 90, 32, torch.float32))
    dirs = [torch.randn_like(x) for x in (q, k, v)]
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = ts.windowed_attention(*leaves, window=25, sinks=2)
    grads = torch.autograd.grad(out, leaves, do)
    slope = sum((g.double() * d.double()).sum() for g, d in zip(grads, dirs))
    h = 2.0 ** -7

    def at(c):
        return (ts.windowed_attention(*(x + c * d for x, d in zip((q, k, v), dirs)), window=25, sinks=2).double() * do).sum()

    diff = (at(h) - at(-h)) / (2 * h)
    # (third derivatives of some 10 times the slope's scale over h^2 / 6, and fp32 outputs of norm 60 over h)
    assert abs(float(slope - diff)) < 1e-3 * float(sum((g * d).norm() for g, d in zip(grads, dirs))) + 1e-3


def test_compiled_and_unrecorded_calls_are_the_same(cuda):
    import thetascan_amd as ts

    q, k, v, do = (x.to(cuda) for x in inputs(2, 4, 2, 150, 64, torch.bfloat16))
    lengths = torch.tensor([150, 77], device=cuda)

    def f(q, k, v):
        return ts.windowed_attention(q, k, v, window=40, sinks=2, lengths=lengths)

    base = f(q, k, v)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = f(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    again = torch.compile(f, fullgraph=True)(*leaves)
    more = torch.autograd.grad(again, leaves, do)
    assert torch.equal(base, out) and torch.equal(out, again)
    assert all(torch.equal(a, b) for a, b in zip(grads, more))
    out = f(*leaves)
    (g,) = torch.autograd.grad(out, leaves[:1], do, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


def test_graphs_replay_with_new_inputs(cuda):
    """A captured training pass, replayed with other inputs and eager work between; another
    stream than the current one."""
    import thetascan_amd as ts

    data = [[x.to(cuda) for x in inputs(2, 4, 2, 300, 64, torch.bfloat16, s)] for s in range(3)]
    leaves = [x.clone().requires_grad_(True) for x in data[0][:3]]
    do = data[0][3].clone()

    def step():
        out = ts.windowed_attention(*leaves, window=70, sinks=20)
        return [out, *torch.autograd.grad(out, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for s in (1, 2, 0):
        with torch.no_grad():
            for x, y in zip([*leaves, do], data[s]):
                x.copy_(y)
        want = [x.detach().clone() for x in step()]
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x.detach(), y)


# ------------------------------------------------------------------ single tokens

@pytest.mark.parametrize("H,Hk,d,window,sinks", [(4, 2, 64, 16, 3), (8, 1, 128, 40, 0), (3, 3, 16, 1, 2), (40, 2, 80, 33, 5),
                                                 (2, 2, 64, 1, 0), (4, 4, 40, 300, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_steps_are_the_sequence(cuda, H, Hk, d, window, sinks, dtype):
    """Token after token from caches that hold NaN: each output within the sequence's bars; after a
    prompt of some length, the same; a free place is left as it is."""
    import thetascan_amd as ts

    T, B = 90, 3
    q, k, v, do = inputs(B, H, Hk, T, d, dtype, d)
    want, bars = reference(q, k, v, do, window, sinks)
    qd, kd, vd = (x.to(cuda) for x in (q, k, v))
    for start in (0, 50):
        caches = [torch.full((B, Hk, sinks + window, d), math.nan, dtype=dtype, device=cuda) for _ in range(2)]
        first = torch.tensor([start, max(start - 7, 0), 0], device=cuda)
        ts.fill_window_cache(kd[:, :, :start], vd[:, :, :start], *caches, sinks=sinks, lengths=first)
        where = first.clone()
        got = torch.full((B, H, T, d), math.nan, dtype=dtype, device=cuda)
        for step in range(T - start):
            at = where.clone()
            at[2] = -1
            rows = [torch.stack([x[b, :, int(min(where[b], T - 1))] for b in range(B)])[:, :, None] for x in (qd, kd, vd)]
            out = ts.windowed_attention_step(*rows, *caches, at, sinks=sinks)
            assert not out[2].any()
            for b in range(2):
                got[b, :, int(at[b])] = out[b, :, 0]
            where += 1
        torch.cuda.synchronize()
        assert torch.isnan(caches[0][2]).all() and torch.isnan(caches[1][2]).all()
        for b in range(2):
            n0, n1 = int(first[b]), int(first[b]) + T - start
            close(f"steps of {b} from {n0}", got[b, :, n0:n1], want[0][b, :, n0:n1], bars[0][b, :, n0:n1])


@pytest.mark.parametrize("B,Hk,window", [(1, 1, 5000), (1, 4, 8192), (70, 8, 700)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_rings_and_large_batches(cuda, B, Hk, window, dtype):
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(1)
    H, d, sinks = 2 * Hk, 64, 4
    slots = sinks + window
    q = torch.randn(B, H, 1, d, generator=g).to(dtype)
    k, v = (torch.randn(B, Hk, 1, d, generator=g).to(dtype) for _ in range(2))
    ck, cv = (torch.randn(B, Hk, slots, d, generator=g).to(dtype) for _ in range(2))
    pos = torch.tensor([(37 + 997 * b) % (3 * window) for b in range(B)])
    pos[0] = 2 ** 40 + 11
    slot = torch.where(pos < sinks, pos, sinks + (pos - sinks) % window)
    K, V = ck.clone(), cv.clone()
    K[torch.arange(B), :, slot], V[torch.arange(B), :, slot] = k[:, :, 0], v[:, :, 0]
    u, scale = U[dtype], d ** -0.5
    Kd, Vd, qd = K.double(), V.double(), q.double().reshape(B, Hk, 2, d)
    s = scale * (qd @ Kd.transpose(2, 3))
    s = s.masked_fill((torch.arange(slots) > pos[:, None])[:, None, None], -math.inf)
    P = torch.softmax(s, -1)
    want = (P @ Vd).reshape(B, H, 1, d)
    e = 2 * (d + 16) * 2.0 ** -24 * float((scale * (qd.abs() @ Kd.abs().transpose(2, 3))).max()) + (slots + 64) * 2.0 ** -23
    bar = u * want.abs() + (u + e) * (P @ Vd.abs()).reshape(B, H, 1, d)
    dk, dv = ck.to(cuda), cv.to(cuda)
    out = ts.windowed_attention_step(q.to(cuda), k.to(cuda), v.to(cuda), dk, dv, pos.to(cuda), sinks=sinks)
    close("step", out, want, bar)
    assert torch.equal(dk.cpu(), K) and torch.equal(dv.cpu(), V)
    # caches that are rows of one buffer, another stream, int32 positions
    both = torch.stack([ck, cv], 3).to(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p32 = (pos % 2 ** 31).to(cuda, torch.int32) if B > 1 else None
        again = ts.windowed_attention_step(q.to(cuda), k.to(cuda), v.to(cuda), both[:, :, :, 0], both[:, :, :, 1],
                                           pos.to(cuda) if p32 is None else p32, sinks=sinks)
    side.synchronize()
    if p32 is None:
        assert torch.equal(out, again)
    else:
        assert torch.equal(out[1:], again[1:])


def test_a_captured_step(cuda):
    """A graph of a step whose positions count up on the device, against eager steps; its writing
    is autograd's change of the caches."""
    import thetascan_amd as ts

    B, H, Hk, d, window, sinks = 2, 4, 2, 64, 9, 2
    q, k, v, _ = (x.to(cuda) for x in inputs(B, H, Hk, 40, d, torch.bfloat16))
    rows = [x[:, :, :1].clone() for x in (q, k, v)]
    mine = [torch.zeros(B, Hk, sinks + window, d, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    pos = torch.zeros(B, dtype=torch.int64, device=cuda)
    version = mine[0]._version
    ts.windowed_attention_step(*rows, *mine, pos, sinks=sinks)
    assert mine[0]._version > version
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ts.windowed_attention_step(*rows, *mine, pos, sinks=sinks)
        pos += 1
    pos.zero_()
    theirs = [torch.zeros_like(x) for x in mine]
    for t in range(40):
        for x, y in zip(rows, (q, k, v)):
            x.copy_(y[:, :, t:t + 1])
        graph.replay()
        want = ts.windowed_attention_step(*rows, *theirs, torch.full((B,), t, device=cuda), sinks=sinks)
        assert torch.equal(out, want)
