"""Low-rank maps by code with enough rows for the largest tiles (64 places, up to rank 64) and for the maps' gradients
in one wavefront a workgroup, against the 64-bit formulas (oracle/decoders_reference.py).

Tiles are that large from 32768 rows on, with 32 rows a code on average.  A code of more than 512
rows has its maps' gradients from several chunks."""
import pytest
import torch

from test_gpu_adapters import TYPES, _check, _inputs
from test_gpu_decoders import BF16, F16, F32, _codes, _gen

pytestmark = pytest.mark.gpu

N = 33001


def _uneven(N, K, seed):
    """Codes of one row, of a tile and a row more, of none and of thousands, the others alike; some rows have no code."""
    codes = _codes((N,), K - 5, seed, none=0.05)
    codes[7], codes[N - 1] = K - 5, K - 4
    codes[100:164], codes[300:365], codes[1000:4000] = K - 3, K - 2, 1
    return codes


# Widths that are whole vectors, at least one, and some that are less; below and above those where the wavefronts
# share the rows' values out (96 values in 32 bits, 192 in 16) and the results' (192 and 384, or half).
WIDTHS = [(64, 48), (200, 392), (64, 392), (59, 33), (201, 391), (201, 33), (3, 391), (201, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,D,E", [(r, *w) for r in (8, 24, 64, 100) for w in WIDTHS])
def test_large_tiles(gpu, dtype, r, D, E):
    K = 41
    _check(gpu, *_inputs(N, K, D, E, r, dtype, seed=r + D + E, base=(r + D) % 2 == 0, codes=_uneven(N, K, r)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,D,E", [(16, 128, 59), (32, 59, 200)])
def test_large_tiles_by_code(gpu, dtype, r, D, E):
    K = 41
    _check(gpu, *_inputs(N, K, D, E, r, dtype, seed=r, codes=_uneven(N, K, r)), by_code=True)
    two = _codes((N // 2, 2), K, seed=r)
    _check(gpu, *_inputs(two.numel(), K, D, E, r, dtype, seed=r, base=False, codes=two), by_code=True, several=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_tiles_of_bad_codes(gpu, dtype):
    K = 41
    codes = _uneven(N, K, 3).long()
    codes[::1000], codes[11], codes[N - 2] = K, -2, 1 << 40
    _check(gpu, *_inputs(N, K, 70, 45, 20, dtype, codes=codes))
    _check(gpu, *_inputs(N, K, 70, 45, 20, dtype, codes=codes, base=False), by_code=True)


def _blocks(dtype, *widths):
    """Workgroups of a code's chunk: blocks of 64 columns in 32 bits, of 128 in 16."""
    return sum(-(-w // (64 if dtype == F32 else 128)) for w in widths)


# One wavefront a workgroup needs 4096 of them: min(rows / 64, codes + chunks) times the blocks of columns (twice that
# above rank 64).
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,D,E", [(4, 0, 0), (16, 1, -1), (24, -3, 3), (32, 0, 0), (64, 1, -5), (100, 0, 0), (128, 3, 2), (16, None, 0),
                                   (33, 0, None)])
def test_maps_gradients_in_one_wavefront(gpu, dtype, r, D, E):
    """Widths of whole blocks and some more or less; None: less than a vector, beside one of 1024 or more."""
    K = 500
    half = 256 if dtype == F32 else 512
    if r > 64:
        half //= 2
    D, E = (3 if w is None else half + w + (half if D is None or E is None else 0) for w in (D, E))
    blocks = _blocks(dtype, D, E) * (2 if r > 64 else 1)
    assert min(N // 64, K + N // 512) * blocks >= 4096
    _check(gpu, *_inputs(N, K, D, E, r, dtype, seed=r, base=False, codes=_uneven(N, K, r)))
