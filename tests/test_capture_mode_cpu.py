"""Refusals of the call that sets a thread's capture mode (no GPU)."""

import ctypes

from torch_spyre_b200 import _lib


def test_refusals():
    exchange = _lib.lib().b200kv_exchange_capture_mode
    assert exchange(None) == 1 and "mode" in _lib.last_error()
    for mode in (-1, 3):
        assert exchange(ctypes.byref(ctypes.c_int32(mode))) == 1 and "mode" in _lib.last_error()
