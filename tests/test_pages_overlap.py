"""CPU: cache_write refuses pools whose rows lie on each other (an expanded tensor's), before any launch."""

import ctypes

import pytest

from kvskip_amd import _native
from test_pages import _write


@pytest.mark.parametrize("kw", [dict(kp_st=0), dict(vp_st=0), dict(kp_st=112), dict(vp_st=64), dict(kp_st=8, format=2)])
def test_refused(kw):
    lib = _native.lib()
    assert lib.kvskip_cache_write(ctypes.byref(_write(N=0)), None) == 0
    assert lib.kvskip_cache_write(ctypes.byref(_write(N=0, **kw)), None) == -1
    assert "must not overlap" in lib.kvskip_last_error().decode()
