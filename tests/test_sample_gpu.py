"""sample_tokens (ts_sample_tokens) against its definition in float64, row by row.

Tokens have to be equal: the weights are whole numbers, of which a float64 exponential may
differ by one in 2^44, and the inputs' random numbers lie anywhere.  Log-probabilities: fp32 terms of
(|y - max| + 8) 2^-23 of themselves (their rounding, the cap's, and the exponential's), a
sum of V terms by lanes, one rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** 44


def capped(z, cap):
    """cap tanh(z / cap) (or z), less the cap where the highest logit is near it: a float64 tanh near
    one is off by 2^-53, which the weights of logits at the cap, whole numbers of 2^-44, can show."""
    if not cap:
        return z
    near = float(z.max().abs()) >= 0.25 * cap
    return -2.0 * cap * torch.sigmoid(-2.0 * z / cap) if near else cap * torch.tanh(z / cap)


def definition(z, u, temperature=1.0, top_k=None, top_p=None, min_p=None, cap=None):
    """Token of one row z (float64, as rounded to its dtype), by the order of its logits."""
    y = torch.where(z == -math.inf, -math.inf, capped(z, cap))
    if temperature == 0:
        temperature, top_k = 1.0, 1
    w = torch.where(z == -math.inf, 0.0, ((y - y.max()) / temperature).exp() * UNIT).round().long()
    order = torch.sort(z, descending=True, stable=True).indices
    if top_k is not None:
        order = order[:max(int(top_k), 1)]
    before = w[order].cumsum(0) - w[order]
    if top_p is not None:
        total = float(w[order].sum())
        order = order[(before == 0) | (before.double() < top_p * total)]
    if min_p is not None:
        order = order[w[order].double() >= min(min_p, 1.0) * UNIT]
    kept = torch.zeros_like(w)
    kept[order] = w[order]
    run = kept.cumsum(0)
    place = min(math.floor(float(u) * float(run[-1])), int(run[-1]) - 1)
    return int((run <= place).sum())


def log_prob(z, token, cap=None):
    y = cap * torch.tanh(z / cap) if cap else z
    y = torch.where(z == -math.inf, -math.inf, y)
    off = y - y.max()
    p = torch.softmax(off, -1)
    far = torch.where(p > 0, p * (off.abs() + 8.0 + (y.abs() if cap else 0.0)), 0.0).sum()
    V = z.numel()
    lp = float(off[token] - torch.logsumexp(off, -1))
    return lp, float(far) * 2.0 ** -23 + (V / 256 + 32) * 2.0 ** -24 + 2.0 ** -24 * abs(lp) + 2.0 ** -23 * (
        float(y.abs().max()) if cap else 0.0)


def check(cuda, z, u, **kw):
    import thetascan_amd as ts

    N = z.shape[0]
    tokens, lps = ts.sample_tokens(z.to(cuda), u.to(cuda), softcap=kw.get("cap"), **{
        n: x.to(cuda) if torch.is_tensor(x) else x for n, x in kw.items() if n != "cap"})
    tokens, lps = tokens.cpu(), lps.cpu()
    for n in range(N):
        one = {name: (float(x[n]) if torch.is_tensor(x) else x) for name, x in kw.items()}
        want = definition(z[n].double(), u[n], **one)
        assert int(tokens[n]) == want, (n, int(tokens[n]), want, one)
        lp, bar = log_prob(z[n].double(), want, kw.get("cap"))
        assert abs(float(lps[n]) - lp) <= bar, (n, float(lps[n]), lp, bar)
    return tokens


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(temperature=3.0), dict(top_k=1), dict(top_k=7),
            dict(top_k=100000), dict(top_p=0.0), dict(top_p=0.5), dict(top_p=0.95), dict(top_p=1.0), dict(min_p=0.05),
            dict(min_p=1.0), dict(temperature=0.6, top_k=40, top_p=0.9, min_p=0.01)]


@pytest.mark.parametrize("kw", SETTINGS, ids=lambda k: "-".join(f"{n}{x}" for n, x in k.items()) or "plain")
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 1024, 5003, 8192, 8193, 50257])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_settings(cuda, V, kw, dtype):
    g = torch.Generator().manual_seed(V)
    N = 6
    z = 3.0 * torch.randn(N, V, generator=g)
    z[torch.rand(N, V, generator=g) < 0.02] = -math.inf
    z[:, V // 2] = 1.0
    check(cuda, z.to(dtype), torch.rand(N, generator=g), **kw)


@pytest.mark.parametrize("cap", [1.0, 30.0, 1e4, 1e20])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_caps(cuda, cap, dtype):
    g = torch.Generator().manual_seed(3)
    z = 20.0 * torch.randn(8, 3001, generator=g)
    z[:, 5] = -math.inf
    z[1, :] = 500.0  # every logit at the cap
    for kw in SETTINGS:
        check(cuda, z.to(dtype), torch.rand(8, generator=g), cap=cap, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_go_to_the_lowest_index(cuda, dtype):
    g = torch.Generator().manual_seed(4)
    V = 20011
    flat = torch.zeros(V)
    signs = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    steps = torch.randint(0, 3, (V,), generator=g).float()
    few = torch.full((V,), -50.0)
    few[[3, 700, 19000]] = 2.0
    z = torch.stack([flat, signs, steps, few, steps * 1e-30, steps * 1e30]).to(dtype)
    u = torch.tensor([0.0, 0.3, 0.999, 0.5, 0.25, 1.0 - 2.0 ** -24])
    for kw in (dict(), dict(top_k=5), dict(top_k=3000), dict(top_p=0.1), dict(top_p=0.37), dict(top_k=9000, top_p=0.5),
               dict(temperature=0.0), dict(temperature=1e6, top_k=12)):
        check(cuda, z, u, **kw)


def test_near_values_in_fp32(cuda):
    """Logits a rounding apart (three levels of keys), and values of every size."""
    g = torch.Generator().manual_seed(5)
    V = 9001
    a = 4.0 + torch.randint(0, 5000, (V,), generator=g).float() * 2.0 ** -21
    b = torch.randint(-2000, 2000, (V,), generator=g).float() * 2.0 ** -140
    c = torch.randn(V, generator=g) * 10.0 ** torch.randint(-30, 2, (V,), generator=g).float()
    d = -1e30 + torch.zeros(V)
    d[77] = 0.0
    z = torch.stack([a, b, c, d])
    u = torch.rand(4, generator=g)
    for kw in (dict(), dict(top_k=100), dict(top_k=4500), dict(top_p=0.3), dict(top_p=0.9), dict(temperature=1e-3, top_p=0.5),
               dict(temperature=50.0, top_k=333, top_p=0.7)):
        check(cuda, z, u, **kw)


@pytest.mark.parametrize("V", [131072, 300001, (1 << 19) - 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_rows(cuda, V, dtype):
    g = torch.Generator().manual_seed(V)
    z = 2.5 * torch.randn(4, V, generator=g)
    z[2] = 0.25
    u = torch.rand(4, generator=g)
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(temperature=0.8, top_k=70000, top_p=0.95, min_p=1e-4)):
        check(cuda, z.to(dtype), u, **kw)


def test_settings_of_every_row(cuda):
    g = torch.Generator().manual_seed(6)
    N, V = 40, 7001
    z = (3.0 * torch.randn(N, V, generator=g)).bfloat16()
    t = torch.rand(N, generator=g) * 2
    t[::9] = 0.0
    k = torch.randint(-2, 300, (N,), generator=g)
    k[::3] = V + 5
    p = torch.rand(N, generator=g)
    p[::4] = 1.5
    p[1::8] = -1.0
    m = torch.rand(N, generator=g) * 0.2
    m[::5] = 2.0
    u = torch.rand(N, generator=g)
    base = check(cuda, z, u, temperature=t, top_k=k, top_p=p, min_p=m)
    # rows of a wider matrix, unaligned, and of more axes; other dtypes of the settings
    import thetascan_amd as ts

    wide = torch.zeros(N, V + 13, dtype=z.dtype)
    wide[:, 5:V + 5] = z
    got = ts.sample_tokens(wide.to(cuda)[:, 5:V + 5].unflatten(0, (8, 5)), u.to(cuda).view(8, 5), temperature=t.to(cuda).view(8, 5),
                           top_k=k.to(cuda, torch.int32).view(8, 5), top_p=p.to(cuda).view(8, 5), min_p=m.to(cuda).view(8, 5))
    assert torch.equal(got[0].cpu().flatten(), base) and got[0].shape == got[1].shape == (8, 5)


def test_rows_without_a_token(cuda):
    import thetascan_amd as ts

    z = torch.randn(6, 2000)
    z[0] = -math.inf
    z[1, 3] = math.nan
    z[2, 1999] = math.inf
    z[3, 1:] = -math.inf
    t = torch.tensor([1.0, 1.0, 1.0, 1.0, -1.0, math.nan])
    for cap in (None, 30.0):
        tokens, lps = ts.sample_tokens(z.to(cuda), torch.full((6,), 0.99, device=cuda), temperature=t.to(cuda), top_p=0.9,
                                       softcap=cap)
        assert tokens.tolist() == [-1, -1, -1, 0, -1, -1]
        assert torch.isnan(lps[[0, 1, 2, 4, 5]]).all() and lps[3] == 0.0
    tokens, lps = ts.sample_tokens(torch.zeros(0, 50, device=cuda), torch.zeros(0, device=cuda))
    assert tokens.shape == lps.shape == (0,)


def test_frequencies_follow_the_probabilities(cuda):
    """Even random numbers of 2^16 rows draw each token as often as its probability says, within one."""
    import thetascan_amd as ts

    n = 1 << 16
    z = torch.tensor([1.0, -2.0, 0.5, 3.0, -math.inf, 2.0], device=cuda)
    u = (torch.arange(n, device=cuda) + 0.5) / n
    tokens, lps = ts.sample_tokens(z.expand(n, 6), u)
    share = torch.bincount(tokens, minlength=6).double() / n
    assert (share - torch.softmax(z.double(), -1)).abs().max() <= 1.0 / n
    assert torch.allclose(lps, torch.log_softmax(z, -1)[tokens], atol=2e-6)


def test_a_captured_draw_and_the_policy_loss(cuda):
    """The log-probabilities are what policy_loss takes: token_log_probs of the same logits."""
    import thetascan_amd as ts

    g = torch.Generator().manual_seed(8)
    z = (3.0 * torch.randn(3, 64, 1024, generator=g)).bfloat16().to(cuda)
    u = torch.rand(3, 64, generator=g).to(cuda)
    zs, us = z[0].clone(), u[0].clone()
    ts.sample_tokens(zs, us, temperature=0.8, top_p=0.9, softcap=30.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, lps = ts.sample_tokens(zs, us, temperature=0.8, top_p=0.9, softcap=30.0)
    for i in (1, 2, 0):
        zs.copy_(z[i])
        us.copy_(u[i])
        graph.replay()
        want, lp = ts.sample_tokens(z[i], u[i], temperature=0.8, top_p=0.9, softcap=30.0)
        assert torch.equal(tokens, want) and torch.equal(lps, lp)
        assert torch.allclose(lps, ts.token_log_probs(z[i], tokens, softcap=30.0), atol=4e-6)
