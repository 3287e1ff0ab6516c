"""Sizes past the operators' limits, past 32 bits among them, are refused with their real size (on tensors without
memory: the checks come before any work)."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from torch_gsplat_bridge_fast import _lib


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _codes(*shape):
    return _meta(*shape, dtype=torch.int32)


def _refused(what, size, f, *args):
    with pytest.raises(ValueError, match=f"{what} are supported, not {size}"):
        f(*args)


@pytest.mark.parametrize("size", [(1 << 28) + 1, (1 << 32) + 7, (1 << 33) + 1])
def test_codes(size):
    _refused("codes", size, gs.lookup_codes, _codes(5), _meta(size, 2))
    _refused("codes", size, gs.code_log_probs, _meta(5, size), _codes(5))
    _refused("codes", size, gs.code_balance, _meta(5, size), _codes(5))
    _refused("codes", size, gs.code_balance, _meta(2, 5, size), _codes(2, 5))


def test_other_axes():
    _refused("codes", (1 << 24) + 1, gs.code_balance, _meta(5, (1 << 24) + 1), _codes(5))
    for size in ((1 << 20) + 1, (1 << 32) + 3):
        _refused("values per code", size, gs.lookup_codes, _codes(5), _meta(4, size))
        _refused("choices per splat", size, gs.code_balance, _meta(2, 9), _codes(2, size))
    for size in (65536, (1 << 32) + 2):
        _refused("images", size, gs.code_balance, _meta(size, 2, 9), _codes(size, 2))


def test_limits_are_taken():
    """At the limits only the device is refused."""
    def only_device(f, *args):
        with pytest.raises(ValueError, match="must be ROCm device tensors"):
            f(*args)
    only_device(gs.lookup_codes, _codes(5), _meta(_lib.MAX_CODES, _lib.MAX_CODE_WIDTH))
    only_device(gs.code_log_probs, _meta(5, _lib.MAX_CODES), _codes(5))
    only_device(gs.code_balance, _meta(_lib.MAX_BALANCE_IMAGES, 2, _lib.MAX_BALANCE_CODES),
                _codes(_lib.MAX_BALANCE_IMAGES, 2, _lib.MAX_CHOICES))
