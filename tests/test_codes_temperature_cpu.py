"""The C ABI's temperatures: those whose reciprocal in base 2 is past the float's range are refused."""
import ctypes

import pytest

from torch_gsplat_bridge_fast import _lib


@pytest.mark.parametrize("T,taken", [(5.1e-39, True), (4.1e-39, False), (3.4e-39, False), (1e-45, False), (1e-30, True), (3e38, True)])
def test_temperature(T, taken):
    L, d = _lib.lib(), ctypes.c_void_p(256)
    m = _lib.ProbsMeta(0, 5, 2, 5, 0, 4, T)  # (no rows: what is taken returns without a launch)
    assert L.gsplat_hip_code_probs_forward(m, d, d, d, d, d, d, None, d, 1 << 30, None) == (0 if taken else 1)
    if not taken:
        assert "temperature" in L.gsplat_hip_last_error().decode()
