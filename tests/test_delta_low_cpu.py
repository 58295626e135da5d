"""The buffer of low halves that a bf16 training call keeps beside its workspace:
its size, and calls without it are refused on the host."""
from __future__ import annotations

import ctypes

from tests.test_delta_cpu import FAKE, desc, io, strided
from thetascan_amd import _lib


def test_low_halves_are_asked_for():
    lib, n, work = _lib.load(), ctypes.c_size_t(), ctypes.c_size_t()
    d = desc(keep=1)
    assert lib.ts_delta_low_bytes(ctypes.byref(d), ctypes.byref(n)) == _lib.TS_OK
    assert n.value == 16 * 2 * 64 * 64 * 2  # as many as the high ones: U and S0 of 16 chunks
    for other in (desc(), desc(keep=1, dtype=_lib.TS_F32)):
        low = ctypes.c_size_t(1)
        assert lib.ts_delta_low_bytes(ctypes.byref(other), ctypes.byref(low)) == _lib.TS_OK and low.value == 0
    assert lib.ts_delta_low_bytes(ctypes.byref(desc(dk=136)), ctypes.byref(n)) == _lib.TS_ERR_NOT_IMPLEMENTED
    lib.ts_delta_workspace_bytes(ctypes.byref(d), ctypes.byref(work))
    grads = _lib.DeltaGrads(strided(), strided(), strided(), strided(), FAKE, FAKE, None, None, None)
    for low in (None, FAKE + 8):
        args = (ctypes.byref(d), ctypes.byref(io(low=low)))
        assert lib.ts_delta_fwd(*args, FAKE, work.value, None) == _lib.TS_ERR_VALUE
        assert b"low halves" in lib.ts_last_error()
        assert lib.ts_delta_bwd(*args, ctypes.byref(grads), FAKE, work.value, FAKE, 1 << 40, None) == _lib.TS_ERR_VALUE
        assert b"low halves" in lib.ts_last_error()
