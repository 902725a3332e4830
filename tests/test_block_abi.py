"""CPU checks of the norms', the feed-forward block's and the recurrence's entry
points: called before InitEngine they return NULL with a reason, clear what they
would fill, and touch no device."""
import ctypes

import pytest

from directcompute_torch_amd import _lib


def test_calls_without_init_fail_cleanly():
    lib = _lib.open_library()
    info = _lib.GPUInfo()
    lib.GetGPUInfo(ctypes.byref(info))
    if info.vendorId != 0:
        pytest.skip("engine already initialised in this process")
    got = [ctypes.c_void_p(1) for _ in range(5)]
    p = [ctypes.byref(g) for g in got]

    def cleared(n):
        assert all(g.value is None for g in got[:n]) and "not initialised" in _lib.last_error(lib)
        for g in got:
            g.value = 1
        lib.ClearLastError()
    assert lib.RmsNorm(None, None, 1, 1, 1e-6, p[0]) is None
    cleared(1)
    lib.RmsNormBackward(None, None, None, None, 1, 1, *p[:2])
    cleared(2)
    assert lib.ResidualNorm(None, None, None, None, None, 1, 1, 0, 1.0, 1e-6, *p[:2]) is None
    cleared(2)
    lib.ResidualNormBackward(None, None, None, None, None, None, None, None, 1, 1, 0, 1.0, *p)
    cleared(5)
    assert lib.GatedMlpForward(None, None, None, None, 1, 1, 1, 1, 0, p[0]) is None
    cleared(1)
    lib.GatedMlpBackward(None, None, None, None, None, None, 1, 1, 1, 1, 0, *p[:4])
    cleared(4)
    assert lib.GatedScanForward(None, None, None, None, 1, 1, 1, p[0]) is None
    cleared(1)
    lib.GatedScanBackward(None, None, None, None, None, None, 1, 1, 1, *p[:3])
    cleared(3)
