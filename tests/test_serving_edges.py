"""Refusals of the serving entries (include/fyodor_hip_serving.h) for data that they read on the host; no GPU."""
import ctypes

import numpy as np
import pytest

from fyodor_amd.hip import ROPE_SCALINGS, Kernels


@pytest.mark.parametrize("scaling", ["none", "linear", "bands", "ramp"])
@pytest.mark.parametrize("bad", [0.0, -0.0, np.nan, np.inf, -np.inf])
def test_rope_factors_refusals(scaling, bad):
    """A factor that gives no frequency is declined, and nothing is written."""
    kernels = Kernels()
    args = dict(scaling=scaling, factor=4.0, original=4096, low=1, high=32)
    factors = np.linspace(1, 2, 32).astype(np.float32)
    f, _ = kernels.rope_frequencies(64, 10000.0, factors=factors, **args)
    assert np.all(np.isfinite(f)) and np.all(f > 0)
    for at in (0, 13, 31):
        wrong = factors.copy()
        wrong[at] = bad
        with pytest.raises(ValueError):
            kernels.rope_frequencies(64, 10000.0, factors=wrong, **args)
        out, magnitude = np.full(32, 7, np.float32), ctypes.c_float(7)
        assert kernels.lib.nya_hip_rope_frequencies(out.ctypes.data, 64, 10000.0, wrong.ctypes.data,
                                                    ROPE_SCALINGS[scaling], 4.0, 4096.0, 1.0, 32.0,
                                                    ctypes.byref(magnitude)) == 1
        assert np.all(out == 7) and magnitude.value == 7
