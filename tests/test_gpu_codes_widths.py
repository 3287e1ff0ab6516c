"""Rows of logits at the widths where the kernels of code_log_probs and code_balance change: whole teams of
2 to 64 lanes with 1 to 4 vectors a lane, one element less and one more, the next whole vector.  The codebook's
gradient where its splats are sorted, and where chunks of them are added up."""
import pytest
import torch

from test_gpu_codes import BF16, F16, F32, _check_balance, _check_lookup, _check_probs, _gen, _logits, _lookup_inputs

pytestmark = pytest.mark.gpu

TEAMS = sorted({lanes * vectors for lanes in (2, 4, 8, 16, 32, 64) for vectors in (1, 2, 3, 4)})


def _widths(vectors, dtype):
    whole = vectors * (4 if dtype == F32 else 8)
    return [whole - 3, whole - 1, whole, whole + 1, whole + (4 if dtype == F32 else 8)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vectors", TEAMS)
def test_probs_widths(gpu, vectors, dtype):
    for K in _widths(vectors, dtype):
        for rows, top in ((67, 1), (9, 4), (3, 0)):
            x = _logits((rows,), K, dtype, seed=K + top, masked=0.1)
            codes = torch.randint(-1, K, (rows,), generator=_gen(K))
            _check_probs(gpu, x, codes, top, T=0.7, what=f"K={K} {dtype} rows={rows} top={top}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vectors", TEAMS)
def test_balance_widths(gpu, vectors, dtype):
    for K in _widths(vectors, dtype):
        for B, G, S in ((1, 131, 1), (2, 5, 2)):
            x = _logits((B, G), K, dtype, seed=K, masked=0.1)
            codes = torch.randint(-1, K, (B, G, S), generator=_gen(K))
            _check_balance(gpu, x, codes, what=f"K={K} {dtype} B={B} G={G}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K", [45, 101, 190, 381, 770, 1533])
def test_widths_of_columns(gpu, dtype, K):
    """Rows that are columns of wider logits: what lies beside a row, NaN here, reaches no result."""

    def columns(x):
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 13), float("nan"), dtype=dtype, device=gpu)
        wide[..., 5:5 + x.shape[-1]] = x.to(gpu)
        return wide[..., 5:5 + x.shape[-1]].detach()

    x = _logits((70,), K, dtype, seed=K, masked=0.1)
    codes = torch.randint(-1, K, (70,), generator=_gen(K))
    _check_probs(gpu, x, codes, 1, what=f"K={K} {dtype}", view=columns)
    _check_probs(gpu, x, codes, 3, what=f"K={K} {dtype}", view=columns)
    _check_balance(gpu, x, codes, what=f"K={K} {dtype}", view=columns)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [1, 3, 4, 5, 8, 16, 17, 31, 33, 64])
def test_lookup_of_many_splats_and_codes(gpu, dtype, D):
    """Narrow rows above the sizes that are not sorted: runs within and over the teams' pieces."""
    _check_lookup(gpu, *_lookup_inputs((30011 + D,), 9001, D, dtype, skew=D % 2 == 0, seed=D), what=f"D={D} {dtype}")


@pytest.mark.parametrize("D,dtype", [(1, F32), (3, F32), (16, F32), (30, BF16), (32, F16), (64, F32), (130, BF16), (513, F32), (1040, F16)])
@pytest.mark.parametrize("N", [255, 511, 2047, 2049, 4100, 8192, 8193, 20001, 65536, 65537])
def test_lookup_of_few_codes(gpu, N, D, dtype):
    """Splats in chunks whose sums are joined: one code of most splats, of all, chunks without any code."""
    codes, book, s, grad = _lookup_inputs((min(N, 9000) if D > 32 else N,), 37, D, dtype, skew=True, seed=N)
    _check_lookup(gpu, codes, book, s, grad, factor=0.5, what=f"N={N} D={D}")
    _check_lookup(gpu, torch.where(torch.arange(len(codes)) > len(codes) // 3, -torch.ones_like(codes), codes), book, None, grad,
                  what=f"N={N} D={D} pruned")
    _check_lookup(gpu, torch.full_like(codes, 36), book, s, grad, what=f"N={N} D={D} one code")
