"""distill_loss without the tail takes the softmax of what the teacher names: any scores, from
those of a sampled token that was unlikely to unnormalised ones (ts_distill_fwd, ts_distill_bwd), against
float64 of the same scores less their highest.  The bars are those of tests/test_distill_gpu.py.
"""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_distill_gpu import close, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,V", [(7, 500), (5, 3001), (16390, 1000), (520, 2600)])
@pytest.mark.parametrize("K", [1, 5, 70])
@pytest.mark.parametrize("g", [None, 2.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_far_from_zero(cuda, N, V, K, g, dtype):
    gen = torch.Generator().manual_seed(V)
    z = (2.0 * torch.randn(N, V, generator=gen)).to(dtype)
    ids = torch.rand(N, V, generator=gen).argsort(-1)[:, :K].contiguous()
    at = torch.tensor([-100.0, -800.0, -1e5, 90.0, 1e4, 0.0])[torch.arange(N) % 6]
    lps = at[:, None] + (2.0 * torch.randn(N, K, generator=gen)).clamp(-6.0, 6.0)
    if K > 1:
        lps[::3, 1] = -math.inf  # (a share of zero)
        ids[::4, -1], lps[::4, -1] = -1, 1e30  # (no token, whatever its score)
    there = torch.where(ids >= 0, lps.double(), -math.inf)
    near = torch.where(ids >= 0, there - there.amax(-1, keepdim=True), 0.0)
    want, bars = reference(z, ids, near.nan_to_num(neginf=-2000.0), None, 1.0, False, None)
    got = run(cuda, z, ids, lps, g=None if g is None else torch.tensor(g), tail=False)
    scale = 1.0 if g is None else g
    close(got, (*want[:2], scale * want[2]), (*bars[:2], scale * bars[2]))


@pytest.mark.parametrize("N,V", [(6, 500), (6, 3001), (16390, 1000)])
@pytest.mark.parametrize("g", [None, 2.0])
def test_rows_without_a_share(cuda, N, V, g):
    """No score above -inf: the softmax is no number, and neither are loss and gradient; no token at all: zeros."""
    gen = torch.Generator().manual_seed(V)
    z = torch.randn(N, V, generator=gen)
    ids = torch.rand(N, V, generator=gen).argsort(-1)[:, :4].contiguous()
    lps = torch.randn(N, 4, generator=gen)
    lps[1], ids[2], lps[3, 1] = -math.inf, -1, math.nan
    _, each, dz = run(cuda, z, ids, lps, g=None if g is None else torch.tensor(g), tail=False)
    bad = torch.zeros(N, dtype=torch.bool)
    bad[[1, 3]] = True
    assert torch.equal(torch.isnan(each), bad) and torch.equal(torch.isnan(dz).all(-1), bad)
    assert torch.equal(torch.isnan(dz).any(-1), bad)
    assert float(each[2]) == 0.0 and not dz[2].any()
