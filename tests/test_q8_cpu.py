"""What the 8-bit cache's entry points refuse before they touch a GPU."""
import ctypes

import numpy as np
import pytest

from leap_b200 import AttentionContext, _native
from leap_b200.attention import _ints, kv_kind, rope_table


def test_unknown_kinds_are_refused():
    lib = _native.lib()
    c, s = rope_table(16, 64)
    fp = ctypes.POINTER(ctypes.c_float)
    d = _native.CtxDesc(1, 0, 8, 4, 64, 16, 1, 0, c.ctypes.data_as(fp), s.ctypes.data_as(fp))
    h = ctypes.c_void_p()
    for kind in (-1, 2):
        assert lib.leap_ctx_create_kv(ctypes.byref(d), kind, ctypes.byref(h)) == _native.LEAP_ERR_INVALID
        assert b"kv kind" in lib.leap_last_error() and not h.value
    assert lib.leap_ctx_create_kv(None, 1, ctypes.byref(h)) == _native.LEAP_ERR_INVALID
    assert lib.leap_engine_set_kv(None, 1) == _native.LEAP_ERR_INVALID
    with pytest.raises(ValueError):
        AttentionContext(1, 8, 4, 64, 16, kv="q4")
    with pytest.raises(ValueError):
        kv_kind("Q8")


def test_null_contexts_are_refused():
    lib = _native.lib()
    bad = _native.LEAP_ERR_INVALID
    assert lib.leap_attn_prefill_packed(None, 0, 0, *[None] * 7) == bad
    assert lib.leap_attn_tree(None, 0, 0, *[None] * 8) == bad
    assert lib.leap_kv_keep(None, 0, *[None] * 4) == bad
    assert lib.leap_kv_read_packed(None, 0, 0, *[None] * 5) == bad
    assert lib.leap_ctx_kv_kind(None, None) == bad


def test_host_arrays():
    a = np.arange(3, dtype=np.int32)
    assert _ints(a, "a", 3) is a
    assert _ints([1, 2], "a").dtype == np.int32
    for x, n in (([1, 2], 3), ([[1], [2]], None)):
        with pytest.raises(ValueError):
            _ints(x, "a", n)
