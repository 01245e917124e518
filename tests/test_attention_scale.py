"""Scales that 32 bits do not hold, at the C entry (which answers before it touches a device)."""
from __future__ import annotations

import ctypes

import pytest

from conftest import load_pkg

pkg = load_pkg()
L = pkg._lib.lib()
ROOM = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(ROOM) + 15) & ~15


@pytest.mark.parametrize("scale", (float("inf"), float("-inf"), float("nan"), 3e38, -2.0 ** 127, 1e300))
def test_c_attend_refuses(scale):
    view = pkg._lib.KVCacheView(AT, AT, AT, AT, 4, 16, 2, 64, 0)
    a = pkg._lib.AttendArgs(cache=ctypes.pointer(view), q=AT, out=AT, block_table=AT, kv_len=AT, T=0, B=1, width=1, n_heads=2)
    assert L.b200lut_attend(ctypes.byref(a), AT, 1 << 30, None) == 0
    a.scale = scale
    assert L.b200lut_attend(ctypes.byref(a), AT, 1 << 30, None) == 1
    assert "scale" in L.b200lut_last_error().decode()
