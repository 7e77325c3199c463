"""The capture-mode swap refuses what is no mode, before anything touches a GPU."""

from __future__ import annotations

import ctypes

import pytest

from gfx950_gluon_tutorials_b200 import _lib


@pytest.mark.parametrize("mode", [-1, 3])
def test_refuses_what_is_no_mode(mode):
    m = ctypes.c_int(mode)
    assert _lib.lib().b2g_exchange_capture_mode(ctypes.byref(m)) == _lib.EINVAL and m.value == mode
    assert _lib.lib().b2g_exchange_capture_mode(None) == _lib.EINVAL
