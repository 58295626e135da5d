"""Refusals of the gated delta rule and the policy loss on the host: wrong shapes,
dtypes and devices before any launch, and the C entry points' own checks (no
device memory is touched: the pointers here are never dereferenced)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import thetascan_amd as ts
from thetascan_amd import _lib


def streams(B=2, Hk=2, H=4, T=10, dk=16, dv=8, dtype=torch.float32):
    return dict(q=torch.zeros(B, Hk, T, dk, dtype=dtype), k=torch.zeros(B, Hk, T, dk, dtype=dtype),
                v=torch.zeros(B, H, T, dv, dtype=dtype), beta=torch.zeros(B, H, T))


def call(**kw):
    s = streams()
    s.update(kw)
    return ts.gated_delta_rule(**s)


def test_delta_rule_refuses_what_it_does_not_take():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        call()
    for bad in (dict(q=z(2, 10, 16)), dict(k=z(2, 2, 10, 8)), dict(v=z(2, 4, 9, 8)), dict(v=z(1, 4, 10, 8)),
                dict(v=z(2, 3, 10, 8), beta=z(2, 3, 10)), dict(beta=z(2, 4, 9)), dict(beta=z(2, 2, 10)),
                dict(beta=z(2, 4, 10, 2)), dict(retention=z(3)), dict(retention=z(2, 4, 9)),
                dict(retention=z(2, 1, 10)), dict(state=z(2, 4, 16, 9)), dict(state=z(2, 2, 16, 8)),
                dict(state=z(2, 4, 16, 8, dtype=torch.bfloat16)), dict(state_out=z(2, 4, 8, 16)),
                dict(lengths=z(3, dtype=torch.int64)), dict(lengths=z(2)),
                dict(k=z(2, 2, 10, 16, dtype=torch.bfloat16)), dict(v=z(2, 4, 10, 0))):
        with pytest.raises(ValueError):
            call(**bad)
    half = torch.float16
    for bad in (dict(retention=z(2, 4, 10, 16)), dict(q=z(2, 2, 10, 136), k=z(2, 2, 10, 136)),
                dict(v=z(2, 4, 10, 520)), dict(beta=z(2, 4, 10, dtype=half)), dict(retention=z(4, dtype=torch.float64)),
                dict(q=z(2, 2, 10, 16, dtype=half), k=z(2, 2, 10, 16, dtype=half), v=z(2, 4, 10, 8, dtype=half))):
        with pytest.raises(NotImplementedError):
            call(**bad)


def test_policy_loss_refuses_what_it_does_not_take():
    def call(**kw):
        s = dict(logits=torch.zeros(5, 7), tokens=torch.zeros(5, dtype=torch.int64), old_log_probs=torch.zeros(5),
                 advantages=torch.zeros(5))
        s.update(kw)
        return ts.policy_loss(**s)

    with pytest.raises(RuntimeError, match="must live on the GPU"):
        call()
    z = torch.zeros
    for bad in (dict(tokens=z(5)), dict(tokens=z(4, dtype=torch.int64)), dict(old_log_probs=z(4)),
                dict(advantages=z(5, 1)), dict(advantages=z(5, dtype=torch.int64)), dict(weights=z(6)), dict(kl=0.1),
                dict(kl=-1.0, ref_log_probs=z(5)), dict(kl=float("nan"), ref_log_probs=z(5)), dict(clip=-0.1),
                dict(clip=(1.5, 0.2)), dict(clip=(0.2, float("nan"))), dict(softcap=0.0), dict(softcap=-3.0),
                dict(softcap=float("inf")), dict(logits=z(5, 0)), dict(kl=0.1, ref_log_probs=z(4))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(NotImplementedError):
        call(logits=z(5, 7, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        ts.token_log_probs(z(5, 7), z(5, dtype=torch.int64))


def test_gated_delta_config():
    with pytest.raises(ValueError):
        ts.GatedDelta(ts.GatedDeltaConfig(d_model=100, n_heads=3))
    with pytest.raises(ValueError):
        ts.GatedDelta(ts.GatedDeltaConfig(d_model=64, n_heads=4, key_heads=3))
    with pytest.raises(NotImplementedError):
        ts.GatedDelta(ts.GatedDeltaConfig(d_model=512, n_heads=2))
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        ts.GatedDelta(ts.GatedDeltaConfig(d_model=64, n_heads=2))(torch.zeros(1, 3, 64))


FAKE = 1 << 20  # 16-byte aligned, never dereferenced


def desc(**kw):
    f = dict(B=2, Hk=2, H=4, T=100, dk=64, dv=64, dtype=_lib.TS_BF16, beta_dtype=_lib.TS_BF16, decay_dtype=_lib.TS_F32,
             keep=0)
    f.update(kw)
    return _lib.DeltaDesc(*f.values())


def strided(st=64, ptr=FAKE):
    return _lib.Strided(ptr, 6400, 64, st)


def io(**kw):
    f = dict(q=strided(), k=strided(), v=strided(), beta=strided(), decay=strided(), out=strided(), lengths=None,
             state=None, state_out=None)
    f.update(kw)
    return _lib.DeltaIO(*f.values())


def test_delta_entry_points_check_on_the_host():
    lib = _lib.load()
    n = ctypes.c_size_t()
    assert lib.ts_delta_workspace_bytes(ctypes.byref(desc()), ctypes.byref(n)) == _lib.TS_OK
    # eight heads x two chunks: two triangles in bf16 pairs (6 fragments of 1 KiB each) and 196 floats
    assert n.value == 16 * (4 * 6 * 1024 + 196 * 4)
    small = n.value
    assert lib.ts_delta_workspace_bytes(ctypes.byref(desc(keep=1)), ctypes.byref(n)) == _lib.TS_OK
    assert n.value == small + 16 * 2 * 64 * 64 * 2  # and what the backward reads: U and S0
    for bad, code in ((dict(dk=136), 2), (dict(dv=520), 2), (dict(dk=60), 1), (dict(dv=4), 1), (dict(H=3), 1),
                      (dict(T=-1), 1), (dict(B=0), 1), (dict(dtype=7), 2)):
        assert lib.ts_delta_workspace_bytes(ctypes.byref(desc(**bad)), ctypes.byref(n)) == code, bad
    call = lib.ts_delta_fwd
    d, work = desc(), ctypes.c_void_p(FAKE)
    assert call(ctypes.byref(d), None, work, small, None) == _lib.TS_ERR_VALUE
    for bad in (dict(q=strided(ptr=FAKE + 2)), dict(v=strided(ptr=None)), dict(out=strided(st=60)),
                dict(beta=strided(ptr=None))):
        assert call(ctypes.byref(d), ctypes.byref(io(**bad)), work, small, None) == _lib.TS_ERR_VALUE, bad
    # 64 rows of a chunk in 2 GiB
    assert call(ctypes.byref(d), ctypes.byref(io(k=strided(st=1 << 24))), work, small, None) == _lib.TS_ERR_NOT_IMPLEMENTED
    assert b"2 GiB" in lib.ts_last_error()
    for ws, size in ((work, small - 1), (ctypes.c_void_p(FAKE + 8), small), (None, small)):
        assert call(ctypes.byref(d), ctypes.byref(io()), ws, size, None) == _lib.TS_ERR_VALUE
    assert b"workspace" in lib.ts_last_error()
    assert lib.ts_delta_step(ctypes.byref(d), ctypes.byref(io(state=FAKE + 4)), None) == _lib.TS_ERR_VALUE
    grads = _lib.DeltaGrads(strided(), strided(), strided(), strided(), FAKE, FAKE, None, None, None)
    assert lib.ts_delta_bwd(ctypes.byref(d), ctypes.byref(io()), ctypes.byref(grads), work, 8, work, 1 << 30,
                            None) == _lib.TS_ERR_VALUE
    assert b"saved" in lib.ts_last_error()


def test_policy_entry_points_check_on_the_host():
    lib = _lib.load()

    def d(**kw):
        f = dict(rows=10, stride=64, V=64, dtype=_lib.TS_BF16, cap=30.0, reserved=0, kl=0.1, low=0.2, high=0.2)
        f.update(kw)
        return _lib.PolicyDesc(*f.values())

    n = ctypes.c_int64()
    assert lib.ts_policy_loss_parts(ctypes.byref(d()), ctypes.byref(n)) == _lib.TS_OK and n.value == 3
    for bad, code in ((dict(rows=-1), 1), (dict(V=0), 1), (dict(cap=-1.0), 1), (dict(low=1.5), 1), (dict(kl=-0.1), 1),
                      (dict(high=float("nan")), 1), (dict(dtype=5), 2), (dict(rows=1 << 32), 2)):
        assert lib.ts_policy_loss_parts(ctypes.byref(d(**bad)), ctypes.byref(n)) == code, bad
    full = _lib.PolicyIO(*[FAKE] * 12)
    for name in ("logits", "tokens", "old_log_probs", "advantages", "log_probs", "coef", "lse", "parts"):
        missing = _lib.PolicyIO(*[None if f[0] == name else FAKE for f in _lib.PolicyIO._fields_])
        assert lib.ts_policy_loss_fwd(ctypes.byref(d()), ctypes.byref(missing), None) == _lib.TS_ERR_VALUE, name
    assert lib.ts_policy_loss_bwd(ctypes.byref(d()), ctypes.byref(full), None, FAKE, None) == _lib.TS_ERR_VALUE
    assert lib.ts_policy_loss_bwd(ctypes.byref(d()), ctypes.byref(full), FAKE, FAKE + 1, None) == _lib.TS_ERR_VALUE


def test_sizes_past_a_launch_are_refused():
    lib, n, m = _lib.load(), ctypes.c_size_t(), ctypes.c_int64()
    for B, code in (((1 << 22) - 1, _lib.TS_OK), (1 << 22, _lib.TS_ERR_NOT_IMPLEMENTED)):
        assert lib.ts_delta_workspace_bytes(ctypes.byref(desc(B=B, T=1)), ctypes.byref(n)) == code
    for V, rows in ((2048, 1 << 26), (2049, 1 << 24)):
        for less, code in ((1, _lib.TS_OK), (0, _lib.TS_ERR_NOT_IMPLEMENTED)):
            d = _lib.PolicyDesc(rows - less, V, V, _lib.TS_BF16, 0.0, 0, 0.0, 0.0, 0.0)
            assert lib.ts_policy_loss_parts(ctypes.byref(d), ctypes.byref(m)) == code


def test_caps_that_fp32_does_not_hold_are_refused():
    z = torch.zeros
    for cap in (1e-50, 1e-40, 1e39):
        with pytest.raises(ValueError, match="softcap"):
            ts.policy_loss(z(5, 7), z(5, dtype=torch.int64), z(5), z(5), softcap=cap)
        with pytest.raises(ValueError, match="softcap"):
            ts.token_log_probs(z(5, 7), z(5, dtype=torch.int64), softcap=cap)
    n = ctypes.c_int64()
    for cap, code in ((1e-40, 1), (1e39, 1), (1e-30, 0), (1e30, 0)):
        d = _lib.PolicyDesc(5, 7, 7, _lib.TS_F32, cap, 0, 0.0, 0.0, 0.0)
        assert _lib.load().ts_policy_loss_parts(ctypes.byref(d), ctypes.byref(n)) == code
