"""What the backward of windowed attention needs and refuses where sinks are many, on the host."""
from __future__ import annotations

import ctypes

from thetascan_amd import _lib

FAKE = 1 << 20  # (never dereferenced: every call here is refused)


def desc(**kw):
    f = dict(B=8, H=8, Hkv=4, T=32768, d=64, dtype=_lib.TS_BF16, window=1024, sinks=8192, scale=0.125)
    f.update(kw)
    return _lib.WindowDesc(*f.values())


def test_scratch_does_not_grow_with_sinks_times_stretches():
    """The sinks' sums in fp32 (8192 rows of two gradients of 64 for 32 heads), by those near them and by one or
    two stretches of the queries behind, and dout . out; some sinks of a long text take what they took."""
    lib, n = _lib.load(), ctypes.c_size_t()
    sums = 8 * 4 * 8192 * 2 * 64 * 4
    assert lib.ts_window_attention_bwd_workspace_bytes(ctypes.byref(desc()), ctypes.byref(n)) == _lib.TS_OK
    assert n.value <= 3 * sums + 8 * 8 * 32768 * 4
    for B, H, Hkv, T, d, window, sinks in ((1, 8, 8, 1 << 20, 128, 64, 100000), (1, 1, 1, 1 << 20, 128, 1, 250000),
                                           (64, 8, 8, 4096, 128, 1, 4096), (1, 8, 1, 8192, 64, 16, 8000)):
        one = desc(B=B, H=H, Hkv=Hkv, T=T, d=d, window=window, sinks=sinks)
        assert lib.ts_window_attention_bwd_workspace_bytes(ctypes.byref(one), ctypes.byref(n)) == _lib.TS_OK
        tokens, wide = B * H * T, B * H * sinks * 2 * d * 4
        # (some 2048 workgroups' stretches of 128 keys at most, beside the near sums and one stretch)
        assert n.value <= 4 * tokens + 16 + 2 * wide + 2048 * 128 * 2 * d * 4 + (
            tokens * 2 * d * 4 if B * Hkv * T < 128 * 128 else 0), (B, T, sinks)


def test_what_the_backward_refuses_the_forward_refuses():
    lib, n = _lib.load(), ctypes.c_size_t()
    row, none = _lib.Strided(FAKE, 0, 0, 64), _lib.Strided(None, 0, 0, 0)
    io = _lib.WindowIO(row, row, row, row, None, FAKE, none)
    grads = _lib.WindowGrads(row, row, row, row)
    for kw in (dict(B=1, T=65535 * 64, sinks=1000, H=1, Hkv=1, d=128), dict(B=1, T=1 << 21, sinks=1 << 20, d=128)):
        one = desc(**kw)
        assert lib.ts_window_attention_bwd_workspace_bytes(ctypes.byref(one), ctypes.byref(n)) == _lib.TS_ERR_NOT_IMPLEMENTED
        assert lib.ts_window_attention_fwd(ctypes.byref(one), ctypes.byref(io), None) == _lib.TS_ERR_NOT_IMPLEMENTED
        assert lib.ts_window_attention_bwd(ctypes.byref(one), ctypes.byref(io), ctypes.byref(grads), FAKE, 1 << 62,
                                           None) == _lib.TS_ERR_NOT_IMPLEMENTED


def test_scales_that_fp32_does_not_hold():
    import pytest
    import torch

    import thetascan_amd as ts

    n = ctypes.c_size_t()
    for scale in (1e-39, 2.4e38, 3e38, float("inf"), float("nan")):
        one = desc(scale=scale)
        assert _lib.load().ts_window_attention_bwd_workspace_bytes(ctypes.byref(one), ctypes.byref(n)) == _lib.TS_ERR_VALUE
        x = torch.zeros(1, 1, 2, 16)
        with pytest.raises(ValueError, match="scale must be positive"):
            ts.windowed_attention(x, x, x, scale=scale)
