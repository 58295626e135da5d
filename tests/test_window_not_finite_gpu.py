"""Gradients of windowed attention where an input holds a value that is not finite: it reaches what
its formula has it in and nothing else (ts_window_attention_bwd).  All others against float64 of the same
inputs without it, by the bars of tests/test_window_gpu.py.
"""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_window_gpu import inputs, reference, run, visible

pytestmark = pytest.mark.gpu


def reached(name, at, seen):
    """Tokens of (out, dq, dk, dv) that a bad value in token `at` of an input reaches."""
    T = seen.shape[0]
    none = torch.zeros(T, dtype=torch.bool)
    if name in "kv":
        queries = seen[:, at].clone()  # the queries that see it
    else:
        queries = none.clone()
        queries[at] = True
    keys = seen[queries].any(0)  # and the keys whose gradients have those
    return (queries if name != "do" else none, queries, keys, none if name == "v" else keys)


@pytest.mark.parametrize("B,H,Hk,T,d", [(1, 2, 2, 200, 64), (1, 4, 2, 331, 128), (1, 3, 1, 200, 16), (8, 8, 4, 577, 64),
                                        (8, 8, 2, 577, 128), (16, 8, 4, 391, 40)])
@pytest.mark.parametrize("window,sinks", [(20, 3), (90, 70)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_who_does_not_meet_it(cuda, B, H, Hk, T, d, window, sinks, dtype):
    q, k, v, do = inputs(B, H, Hk, T, d, dtype, d)
    rep, seen = H // Hk, visible(T, window, sinks)
    want, bars = reference(*(x[:1] for x in (q, k, v, do)), window, sinks)
    for case, at in enumerate((0, 2, 70, 130, T - 1)):
        for name in ("k", "v", "q", "do"):
            bad = (math.nan, math.inf, -math.inf)[case % 3]
            x = {"q": q.clone(), "k": k.clone(), "v": v.clone(), "do": do.clone()}
            x[name][0, 0, at, 5] = bad
            got = run(cuda, x["q"], x["k"], x["v"], x["do"], window=window, sinks=sinks)
            mask = reached(name, at, seen)
            for what, y, w, bar, hit in zip(("out", "dq", "dk", "dv"), got, want, bars, mask):
                y = y.detach()[:1].double().cpu()
                there = torch.zeros(y.shape[:3], dtype=torch.bool)
                heads = slice(0, rep if what in ("out", "dq") and name in "kv" else 1)
                there[0, heads] = hit
                err = torch.where(there[..., None], 0.0, (y - w).abs())
                worst = float((err / bar).max())
                assert worst <= 1.0, (name, at, bad, what, worst)
                if math.isnan(bad) and name != "v" and what != "out":
                    assert not torch.isfinite(y[there]).all(-1).any(), (name, at, what)
