"""Workspaces stay small beside what a call reads: sums of columns that workgroups leave behind are taken over eight
rows at least above 16384 codes (4 bytes a code: an eighth of the logits in 32 bits, a quarter in 16), and an image's
counts are 4 bytes a code."""
import pytest

from torch_gsplat_bridge_fast import _lib


@pytest.mark.parametrize("batch", [1, 3, 64, 300, 2000])
@pytest.mark.parametrize("rows", [8, 37, 100, 256, 1342, 5000])
@pytest.mark.parametrize("K", [16385, 32768, 100000])
@pytest.mark.parametrize("dtype", [0, 1])
def test_balance_of_long_rows(batch, rows, K, dtype):
    logits = batch * rows * K * (4 if dtype == 0 else 2)
    need = _lib.lib().gsplat_hip_code_balance_workspace_bytes(_lib.BalanceMeta(rows, batch, K, 1, dtype, K, 4))
    # (loss parts, totals and tickets: 16 bytes an image and 4 per 32 codes; parts start on 256 bytes)
    small = batch * (16 + 4 + 4 * (K // 32 + 1)) + 5 * 256
    assert 0 < need <= logits / (8 if dtype == 0 else 4) + 4 * batch * K + small
