"""What sample_tokens and distill_loss refuse, on the host."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import thetascan_amd as ts
from thetascan_amd import _lib

Z, U = torch.zeros(3, 50), torch.zeros(3)


@pytest.mark.parametrize("change,error,match", [
    (dict(logits=torch.zeros(())), ValueError, "logits must be"),
    (dict(logits=torch.zeros(3, 0)), ValueError, "logits must be"),
    (dict(logits=torch.zeros(3, 1).expand(3, 1 << 19)), NotImplementedError, "at most"),
    (dict(logits=Z.half()), NotImplementedError, "bfloat16 or float32"),
    (dict(uniforms=torch.zeros(2)), ValueError, "uniforms must be"),
    (dict(uniforms=torch.zeros(3, dtype=torch.int64)), ValueError, "uniforms must be"),
    (dict(temperature=-0.1), ValueError, "temperature must be"),
    (dict(temperature=float("nan")), ValueError, "temperature must be"),
    (dict(temperature=torch.zeros(2)), ValueError, "temperature must be"),
    (dict(temperature=torch.zeros(3, dtype=torch.int64)), ValueError, "temperature must be"),
    (dict(top_k=0), ValueError, "top_k must be"),
    (dict(top_k=2.0), ValueError, "top_k must be"),
    (dict(top_k=True), ValueError, "top_k must be"),
    (dict(top_k=torch.zeros(3)), ValueError, "top_k must be"),
    (dict(top_p=-1.0), ValueError, "top_p must be"),
    (dict(min_p=float("inf")), ValueError, "min_p must be"),
    (dict(softcap=0.0), ValueError, "softcap must be"),
    (dict(softcap=float("nan")), ValueError, "softcap must be"),
    (dict(), RuntimeError, "must live on the GPU"),
])
def test_sampling_refuses(change, error, match):
    with pytest.raises(error, match=match):
        ts.sample_tokens(**{"logits": Z, "uniforms": U, **change})


IDS, LPS = torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4)


@pytest.mark.parametrize("change,error,match", [
    (dict(logits=torch.zeros(3, 0)), ValueError, "logits must be"),
    (dict(logits=torch.zeros(3, 1).expand(3, (1 << 20) + 1)), NotImplementedError, "at most"),
    (dict(logits=Z.half()), NotImplementedError, "bfloat16 or float32"),
    (dict(ids=IDS[:2]), ValueError, "ids must be"),
    (dict(ids=IDS[:, 0]), ValueError, "ids must be"),
    (dict(ids=IDS[:, :0]), ValueError, "ids must be"),
    (dict(ids=IDS.int()), ValueError, "ids must be"),
    (dict(log_probs=LPS[:, :3]), ValueError, "log_probs must be"),
    (dict(log_probs=IDS), ValueError, "log_probs must be"),
    (dict(weights=torch.zeros(4)), ValueError, "weights must be"),
    (dict(temperature=0.0), ValueError, "temperature must lie"),
    (dict(temperature=float("nan")), ValueError, "temperature must lie"),
    (dict(softcap=-1.0), ValueError, "softcap must be"),
    (dict(), RuntimeError, "must live on the GPU"),
])
def test_distillation_refuses(change, error, match):
    with pytest.raises(error, match=match):
        ts.distill_loss(**{"logits": Z, "ids": IDS, "log_probs": LPS, **change})


def test_tangents_are_refused():
    with forward_ad.dual_level():
        z = forward_ad.make_dual(Z, torch.ones_like(Z))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ts.distill_loss(z, IDS, LPS)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ts.sample_tokens(z, U)


def test_the_library_refuses_by_itself():
    """The C entry points' own checks; the pointers here are never dereferenced."""
    lib, fake = _lib.load(), 1 << 20

    def sample(desc=None, **kw):
        d = dict(rows=3, stride=50, V=50, dtype=_lib.TS_F32, cap=0.0, reserved=0, temperature=1.0, top_p=1.0, min_p=0.0,
                 top_k=50)
        d.update(desc or {})
        names = [n for n, _ in _lib.SampleIO._fields_]
        io = _lib.SampleIO(*(kw.get(n, fake) for n in names))
        return lib.ts_sample_tokens(ctypes.byref(_lib.SampleDesc(*d.values())), ctypes.byref(io), None)

    for bad in (dict(rows=-1), dict(V=0), dict(cap=-1.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(top_p=-0.5), dict(min_p=float("nan")), dict(top_k=0), dict(stride=-1)):
        assert sample(bad) == _lib.TS_ERR_VALUE, bad
    for bad in (dict(V=1 << 19), dict(dtype=7), dict(rows=1 << 22)):
        assert sample(bad) == _lib.TS_ERR_NOT_IMPLEMENTED, bad
    for bad in (dict(logits=None), dict(logits=fake + 2), dict(uniforms=None), dict(tokens=None), dict(log_probs=None)):
        assert sample(**bad) == _lib.TS_ERR_VALUE, bad
    assert sample(dict(rows=0)) == _lib.TS_OK

    def call(**kw):
        return lib.ts_distill_fwd(ctypes.byref(desc(**kw)), ctypes.byref(io()), None)

    def desc(**kw):
        d = dict(rows=3, stride=50, V=50, K=4, dtype=_lib.TS_F32, tail=1, cap=0.0, aligned=0, temperature=1.0)
        d.update(kw)
        return _lib.DistillDesc(*d.values())

    def io(**kw):
        return _lib.DistillIO(*(kw.get(n, fake) for n, _ in _lib.DistillIO._fields_))

    for bad in (dict(rows=-1), dict(V=0), dict(K=0), dict(cap=-1.0), dict(temperature=0.0), dict(temperature=float("nan"))):
        assert call(**bad) == _lib.TS_ERR_VALUE, bad
    for bad in (dict(V=(1 << 20) + 1), dict(dtype=7), dict(rows=1 << 24)):
        assert call(**bad) == _lib.TS_ERR_NOT_IMPLEMENTED, bad
    for bad in (dict(logits=None), dict(logits=fake + 2), dict(ids=None), dict(log_probs=None), dict(each=None),
                dict(parts=None), dict(loss=None)):
        assert lib.ts_distill_fwd(ctypes.byref(desc()), ctypes.byref(io(**bad)), None) == _lib.TS_ERR_VALUE, bad
    assert lib.ts_distill_fwd(ctypes.byref(desc(aligned=1)), ctypes.byref(io()), None) == _lib.TS_ERR_VALUE  # 50 apart
    assert lib.ts_distill_fwd(ctypes.byref(desc()), ctypes.byref(io(dlogits=fake + 4)), None) == _lib.TS_ERR_VALUE
    for bad in (dict(stats=None), dict(logits=None)):
        assert lib.ts_distill_bwd(ctypes.byref(desc()), ctypes.byref(io(**bad)), fake, fake, None) == _lib.TS_ERR_VALUE, bad
    assert lib.ts_distill_bwd(ctypes.byref(desc()), ctypes.byref(io()), None, fake, None) == _lib.TS_ERR_VALUE
    assert lib.ts_distill_bwd(ctypes.byref(desc()), ctypes.byref(io()), fake, fake + 2, None) == _lib.TS_ERR_VALUE
