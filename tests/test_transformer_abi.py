"""CPU checks of the transformer entry points: called before InitEngine they
return NULL / false with a reason and touch no device."""
import ctypes

import pytest

from directcompute_torch_amd import _lib


def test_calls_without_init_fail_cleanly():
    lib = _lib.open_library()
    info = _lib.GPUInfo()
    lib.GetGPUInfo(ctypes.byref(info))
    if info.vendorId != 0:
        pytest.skip("engine already initialised in this process")
    assert lib.RotaryApply(None, None, None, 1, 1, 1, 2, 2, 0) is None
    st = ctypes.c_void_p(1)
    assert lib.AttentionForward(None, None, None, None, 1, 1, 1, 1, 1, 1, 0, 1.0, ctypes.byref(st)) is None
    assert st.value is None and "not initialised" in _lib.last_error(lib)
    got = [ctypes.c_void_p(1) for _ in range(3)]
    lib.AttentionBackward(None, None, None, None, None, None, None, 1, 1, 1, 1, 1, 1, 0, 1.0, 1, 1, 1,
                          *[ctypes.byref(p) for p in got])
    assert all(p.value is None for p in got)
    assert not lib.MuonBatch(None, None, None, None, None, None, 1, 0.9, 1, 0.0, 1.0, 5)
