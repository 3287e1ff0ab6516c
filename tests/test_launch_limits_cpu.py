"""A launch of 2^32 threads and more is refused before it reaches the runtime, which would cut it silently."""
import ctypes

import pytest

from torch_gsplat_bridge_fast import _lib


@pytest.mark.parametrize("width", [1 << 10, 1 << 20])
def test_launch_of_too_many_threads(width):
    """An output of 2^41 bytes and more: 2^27 workgroups of 256 threads at least."""
    L, d = _lib.lib(), ctypes.c_void_p(256)
    m = _lib.LookupMeta(1 << 29, 5, width, width, 0, 4, 1.0)
    assert L.gsplat_hip_lookup_forward(m, d, d, None, d, None) == 2
    text = L.gsplat_hip_last_error().decode()
    assert "lookup_fwd_kernel" in text and "2^32 threads" in text
    # (and the next call is not blamed for it)
    assert L.gsplat_hip_lookup_forward(None, d, d, None, d, None) == 1
    assert "meta is NULL" in L.gsplat_hip_last_error().decode()
