"""What windowed attention, its step and its cache refuse, on the host."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import thetascan_amd as ts
from thetascan_amd import _lib


def streams(H=4, Hk=2, T=10, d=16, dtype=torch.float32):
    return dict(q=torch.zeros(2, H, T, d, dtype=dtype), k=torch.zeros(2, Hk, T, d, dtype=dtype),
                v=torch.zeros(2, Hk, T, d, dtype=dtype))


def ring(d=16, slots=9, dtype=torch.float32):
    return dict(cache_k=torch.zeros(2, 2, slots, d, dtype=dtype), cache_v=torch.zeros(2, 2, slots, d, dtype=dtype))


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(4, 10, 16)), ValueError, "q must be"),
    (dict(k=torch.zeros(2, 2, 9, 16)), ValueError, "do not match"),
    (dict(v=torch.zeros(2, 2, 10, 8)), ValueError, "do not match"),
    (dict(q=torch.zeros(2, 3, 10, 16)), ValueError, "3 query heads over 2"),
    (dict(v=torch.zeros(2, 2, 10, 16, dtype=torch.bfloat16)), ValueError, "one dtype"),
    (dict(window=0), ValueError, "window must be"),
    (dict(window=2.0), ValueError, "window must be"),
    (dict(window=True), ValueError, "window must be"),
    (dict(sinks=-1), ValueError, "sinks must be"),
    (dict(scale=0.0), ValueError, "scale must be"),
    (dict(scale=float("nan")), ValueError, "scale must be"),
    (dict(scale=float("inf")), ValueError, "scale must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError, "lengths must be"),
    (dict(lengths=torch.zeros(2)), ValueError, "lengths must be"),
    (dict(), RuntimeError, "must live on the GPU"),
    (streams(dtype=torch.float16), NotImplementedError, "bfloat16 or float32"),
    (streams(d=136), NotImplementedError, "at most 128"),
    (streams(H=0, Hk=0), ValueError, "heads"),
])
def test_attention_refuses(change, error, match):
    with pytest.raises(error, match=match):
        ts.windowed_attention(**{**streams(), **change})


@pytest.mark.parametrize("change,error,match", [
    (streams(T=2), ValueError, "one token"),
    (dict(sinks=9), ValueError, "9 of them sinks"),
    (dict(cache_v=torch.zeros(2, 2, 8, 16)), ValueError, "slots"),
    (dict(cache_k=torch.zeros(2, 4, 9, 16)), ValueError, "cache_k must be"),
    (dict(cache_k=torch.zeros(2, 2, 9, 16, dtype=torch.bfloat16)), ValueError, "cache_k must be"),
    (dict(cache_k=torch.zeros(1, 2, 9, 16).expand(2, -1, -1, -1)), ValueError, "rows of its own"),
    (dict(cache_v=torch.zeros(2, 2, 9, 18)[..., :16]), ValueError, "rows of its own"),
    (dict(cache_v=torch.zeros(2, 2, 16, 9).transpose(2, 3)), ValueError, "rows of its own"),
    (dict(cache_k=torch.zeros(2, 2, 9, 16, requires_grad=True)), ValueError, "no part in gradients"),
    (dict(q=torch.zeros(2, 4, 1, 16, requires_grad=True)), ValueError, "no part in gradients"),
    (dict(positions=torch.zeros(2)), ValueError, "positions must be"),
    (dict(positions=torch.zeros(1, dtype=torch.int64)), ValueError, "positions must be"),
    ({**streams(T=1, d=18), **ring(18)}, NotImplementedError, "16-byte"),
    (dict(), RuntimeError, "must live on the GPU"),
])
def test_step_refuses(change, error, match):
    args = {**streams(T=1), **ring(), "positions": torch.zeros(2, dtype=torch.int64), "sinks": 2, **change}
    with pytest.raises(error, match=match):
        ts.windowed_attention_step(**args)


def test_one_cache_for_both_is_refused():
    one = torch.zeros(2, 2, 9, 16)
    s = streams(T=1)
    with pytest.raises(ValueError, match="a cache each"):
        ts.windowed_attention_step(**s, cache_k=one, cache_v=one, positions=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="a cache each"):
        ts.fill_window_cache(s["k"], s["v"], one, one)
    with pytest.raises(ValueError, match="lengths must be"):
        ts.fill_window_cache(s["k"], s["v"], **ring(), lengths=torch.zeros(2))
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        ts.fill_window_cache(s["k"], s["v"], **ring())


def test_tangents_are_refused():
    for name in "qkv":
        s = streams()
        with forward_ad.dual_level():
            s[name] = forward_ad.make_dual(s[name], torch.ones_like(s[name]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ts.windowed_attention(**s)


def test_the_library_refuses_by_itself():
    """The C entry points' own checks; the pointers here are never dereferenced."""
    lib, n, fake = _lib.load(), ctypes.c_size_t(), 1 << 20

    def desc(**kw):
        f = dict(B=1, H=4, Hkv=2, T=300, d=64, dtype=_lib.TS_BF16, window=64, sinks=4, scale=0.125)
        f.update(kw)
        return _lib.WindowDesc(*f.values())

    def bytes_of(**kw):
        return lib.ts_window_attention_bwd_workspace_bytes(ctypes.byref(desc(**kw)), ctypes.byref(n))

    row, none = _lib.Strided(fake, 0, 0, 64), _lib.Strided(None, 0, 0, 0)
    io = _lib.WindowIO(row, row, row, row, None, fake, none)
    assert bytes_of() == _lib.TS_OK and n.value >= 4 * 300 * 4
    for bad in (dict(H=3), dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(scale=float("inf")), dict(T=-1), dict(B=0)):
        assert bytes_of(**bad) == _lib.TS_ERR_VALUE, bad
    for bad in (dict(d=136), dict(d=60), dict(dtype=5), dict(T=2 ** 31 - 1), dict(B=2 ** 24)):
        assert bytes_of(**bad) == _lib.TS_ERR_NOT_IMPLEMENTED, bad
    odd = _lib.WindowIO(row, _lib.Strided(fake + 8, 0, 0, 64), row, row, None, fake, none)
    assert lib.ts_window_attention_fwd(ctypes.byref(desc()), ctypes.byref(odd), None) == _lib.TS_ERR_VALUE
    odd = _lib.WindowIO(row, row, _lib.Strided(fake, 0, 0, 65), row, None, fake, none)
    assert lib.ts_window_attention_fwd(ctypes.byref(desc()), ctypes.byref(odd), None) == _lib.TS_ERR_VALUE
    assert lib.ts_window_attention_fwd(ctypes.byref(desc()), None, None) == _lib.TS_ERR_VALUE
    grads = _lib.WindowGrads(row, row, row, row)
    call = lib.ts_window_attention_bwd
    bytes_of()
    assert call(ctypes.byref(desc()), ctypes.byref(io), ctypes.byref(grads), fake, n.value - 1, None) == _lib.TS_ERR_VALUE
    assert call(ctypes.byref(desc()), ctypes.byref(io), ctypes.byref(grads), fake + 8, n.value, None) == _lib.TS_ERR_VALUE
    assert call(ctypes.byref(desc()), ctypes.byref(io), None, fake, n.value, None) == _lib.TS_ERR_VALUE
    bare = _lib.WindowIO(row, row, row, row, None, None, none)
    assert call(ctypes.byref(desc()), ctypes.byref(bare), ctypes.byref(grads), fake, n.value, None) == _lib.TS_ERR_VALUE
    assert lib.ts_window_step_workspace_bytes(ctypes.byref(desc(window=2 ** 31 - 1)), ctypes.byref(n)) == _lib.TS_ERR_NOT_IMPLEMENTED
    assert lib.ts_window_step_workspace_bytes(ctypes.byref(desc()), ctypes.byref(n)) == _lib.TS_OK
    if n.value:
        assert lib.ts_window_step(ctypes.byref(desc()), ctypes.byref(io), row, row, fake, fake, n.value - 1,
                                  None) == _lib.TS_ERR_VALUE
    assert lib.ts_window_step(ctypes.byref(desc()), ctypes.byref(io), row, row, None, fake, n.value, None) == _lib.TS_ERR_VALUE
    off = _lib.Strided(fake + 2, 0, 0, 64)
    assert lib.ts_window_cache_fill(ctypes.byref(desc()), ctypes.byref(io), off, row, None) == _lib.TS_ERR_VALUE
