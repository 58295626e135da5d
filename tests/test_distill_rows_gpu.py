"""distill_loss of many rows, of which a wave takes several (ts_distill_fwd, ts_distill_bwd),
against the definition in float64, in every element of loss and gradient: vocabularies around the sizes at
which a wave's registers hold a row, rows that begin at no 16-byte boundary, rows of weight zero among
others, a last wave with few rows.  The bars are those of tests/test_distill_gpu.py.
"""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_distill_gpu import reference

pytestmark = pytest.mark.gpu


def rows(x, stride, first):
    """``x`` as rows `stride` apart in a buffer of NaN, from its element `first` on."""
    N, V = x.shape
    flat = torch.full((first + N * stride + 8,), math.nan, dtype=x.dtype, device=x.device)
    flat = flat[first:first + (N - 1) * stride + V].as_strided((N, V), (stride, 1))
    return flat.copy_(x)


def check(cuda, N, V, K, dtype, stride=None, first=0, tail=True, cap=None, temperature=1.0, g=None):
    import thetascan_amd as ts

    gen = torch.Generator(device=cuda).manual_seed(V + K + first)
    z = (2.5 * torch.randn(N, V, generator=gen, device=cuda)).to(dtype)
    y = (z.float() + 0.5 * torch.randn(N, V, generator=gen, device=cuda)) / temperature
    lps, ids = torch.log_softmax(y, -1).topk(K, -1)
    weights = torch.rand(N, generator=gen, device=cuda) + 0.5
    weights[torch.rand(N, generator=gen, device=cuda) < 0.3] = 0.0
    weights[-1], weights[-2] = 0.75, 0.0
    weights /= weights.sum()
    with torch.device(cuda):  # (the definition's own tensors beside the inputs)
        want, bars = reference(z, ids, lps, weights, temperature, tail, cap)
    z[weights == 0] = math.nan
    leaf = (z if stride is None else rows(z, stride, first)).requires_grad_(True)
    # (what an unwritten gradient would hold)
    junk = torch.full((N, V), math.nan, dtype=dtype, device=cuda)
    del junk
    loss, each = ts.distill_loss(leaf, ids, lps, weights=weights, tail=tail, softcap=cap, temperature=temperature)
    (dz,) = torch.autograd.grad(loss, leaf, None if g is None else torch.tensor(g, device=cuda))
    scale = 1.0 if g is None else g
    for name, x, y, bar in zip(("loss", "each", "dz"), (loss.detach(), each, dz), (*want[:2], scale * want[2]),
                               (*bars[:2], abs(scale) * bars[2])):
        worst = float(((x.double() - y).abs() / bar.clamp(min=1e-45)).max())
        print(f"{N} x {V}, {K} tokens, {dtype}, {name}: {worst:.3f} of its bar", flush=True)
        assert worst <= 1.0, name
    assert not dz[weights == 0].any() and not each[weights == 0].any()


@pytest.mark.parametrize("V", [1017, 1018, 1019, 1020, 1021, 1022, 1023, 1024, 1025, 2040, 2041, 2047, 2048])
@pytest.mark.parametrize("K", [1, 64, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_vocabularies_at_the_edges(cuda, V, K, dtype):
    check(cuda, 16384, V, K, dtype)


@pytest.mark.parametrize("V", [1016, 1017, 1018, 1021, 1022, 1024, 2043, 2048])
@pytest.mark.parametrize("more,first", [(0, 1), (8, 3), (5, 0), (1, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_begin_anywhere(cuda, V, more, first, dtype):
    check(cuda, 16387, V, 20, dtype, V + more, first)


@pytest.mark.parametrize("N,V,K", [(16391, 1024, 20), (16391, 1000, 100), (16385, 1500, 256), (16399, 64, 64), (16384, 2, 1),
                                   (16390, 8, 3), (16391, 2100, 20)])
@pytest.mark.parametrize("tail,cap,temperature", [(True, None, 1.0), (False, 30.0, 2.0), (True, 5.0, 0.5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forms_of_many_rows(cuda, N, V, K, tail, cap, temperature, dtype):
    check(cuda, N, V, K, dtype, tail=tail, cap=cap, temperature=temperature)


@pytest.mark.parametrize("V,more,first", [(1024, 0, 0), (1023, 0, 0), (1024, 3, 5), (1999, 0, 0)])
@pytest.mark.parametrize("g", [-3.0, 0.25])
def test_other_upstream_gradients(cuda, V, more, first, g):
    """The backward's own kernel, from what the forward keeps of each row."""
    check(cuda, 16391, V, 33, torch.bfloat16, V + more, first, g=g)
    check(cuda, 16391, V, 33, torch.float32, V + more, first, tail=False, g=g)
