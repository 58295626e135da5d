"""Windowed attention, its caches, sampling and distillation on tensors of more than 2^31 elements:
what lies at their ends is as the same call's on that part alone."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_long_batch_of_attention(cuda):
    """[9,32,65536,128] bf16 queries: the last sequence's outputs and gradients, bit for bit (its workgroups
    are as many as the kernels' forms ask for).  The sinks' queries are cut into stretches by the workgroups of
    all sequences, so that their fp32 sums have another order: a step of the rounding, 2^-7 of a value, and
    of the 65536 x 8 terms' sums 2^-24 of their root for each of some 20 additions on a way."""
    import thetascan_amd as ts

    B, H, Hk, T, d = 9, 32, 4, 65536, 128
    g = torch.Generator(device=cuda).manual_seed(1)
    q, do = (torch.randn(B, T, H, d, generator=g, device=cuda, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    k, v = (torch.randn(B, T, Hk, d, generator=g, device=cuda, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    assert q.numel() > 2 ** 31

    def run(*x):
        leaves = [y.detach().requires_grad_(True) for y in x[:3]]
        out = ts.windowed_attention(*leaves, window=64, sinks=4)
        return [out.detach(), *torch.autograd.grad(out, leaves, x[3])]

    got = [x[-1:].clone() for x in run(q, k, v, do)]
    want = run(*(x[-1:] for x in (q, k, v, do)))
    torch.cuda.synchronize()
    for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
        if name in ("dk", "dv"):
            assert torch.allclose(x[:, :, :4].float(), y[:, :, :4].float(), rtol=2.0 ** -7, atol=20 * 2.0 ** -24 * 724.0), name
            x, y = x[:, :, 4:], y[:, :, 4:]
        assert torch.equal(x, y), name


def test_a_long_cache(cuda):
    """[40,8,65540,128] bf16 caches: filled, and read by a step, in the last sequence as in float64."""
    import thetascan_amd as ts

    B, Hk, d, window, sinks, T = 40, 8, 128, 65536, 4, 70000
    g = torch.Generator(device=cuda).manual_seed(2)
    ck, cv = (torch.zeros(B, Hk, sinks + window, d, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    assert ck.numel() > 2 ** 31
    k, v = (torch.randn(1, Hk, T, d, generator=g, device=cuda, dtype=torch.bfloat16).expand(B, -1, -1, -1) for _ in range(2))
    lengths = torch.full((B,), 100, device=cuda)
    lengths[-1] = T
    ts.fill_window_cache(k, v, ck, cv, sinks=sinks, lengths=lengths)
    kept = torch.cat([torch.arange(sinks), torch.arange(T - window, T)]).to(cuda)
    slot = torch.where(kept < sinks, kept, sinks + (kept - sinks) % window)
    for cache, x in ((ck, k), (cv, v)):
        assert torch.equal(cache[-1][:, slot], x[-1][:, kept])
        assert torch.equal(cache[3][:, :100], x[3][:, :100]) and not cache[3][:, 100:].any()
    q = torch.randn(B, Hk, 1, d, generator=g, device=cuda, dtype=torch.bfloat16)
    new = [torch.randn(B, Hk, 1, d, generator=g, device=cuda, dtype=torch.bfloat16) for _ in range(2)]
    out = ts.windowed_attention_step(q, *new, ck, cv, lengths, sinks=sinks)
    at = sinks + (T - sinks) % window
    assert torch.equal(ck[-1][:, at], new[0][-1, :, 0]) and torch.equal(cv[-1][:, at], new[1][-1, :, 0])
    P = torch.softmax((ck[-1].double() * q[-1].double()).sum(-1) * d ** -0.5, -1)
    want = (P[..., None] * cv[-1].double()).sum(1)
    # (65540 alike shares: sums of their roundings, half a step of 2^-9 each, and the output's)
    bar = 2.0 ** -8 * want.abs() + 2.0 ** -8 * (P[..., None] * cv[-1].double().abs()).sum(1)
    assert ((out[-1, :, 0].double() - want).abs() <= bar).all()


def test_many_long_rows_of_logits(cuda):
    """[65700, 32800] bf16: the last rows' losses, gradients and tokens, bit for bit."""
    import thetascan_amd as ts

    N, V, K, last = 65700, 32800, 8, 600
    g = torch.Generator(device=cuda).manual_seed(3)
    z = torch.randn(N, V, generator=g, device=cuda, dtype=torch.bfloat16)
    assert z.numel() > 2 ** 31
    ids = torch.arange(K, device=cuda) * 4001 + torch.arange(N, device=cuda)[:, None] % 4000
    lps = torch.log_softmax(torch.randn(N, K, generator=g, device=cuda), -1) - 0.25
    weights = torch.rand(N, generator=g, device=cuda)

    def run(z, ids, lps, weights):
        leaf = z.detach().requires_grad_(True)
        loss, each = ts.distill_loss(leaf, ids, lps, weights=weights)
        (dz,) = torch.autograd.grad(loss, leaf)
        return each[-last:].clone(), dz[-last:].clone()

    got = run(z, ids, lps, weights)
    want = run(*(x[-last:] for x in (z, ids, lps, weights)))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    u = torch.rand(N, generator=g, device=cuda)
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9)):
        got = [x[-last:] for x in ts.sample_tokens(z, u, **kw)]
        want = ts.sample_tokens(z[-last:], u[-last:], **kw)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
