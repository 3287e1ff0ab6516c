"""Calls whose rows are more than one launch has threads for (2^32 of them), and sizes past 32 bits."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import codes_reference as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _room(gib):
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0] / 2 ** 30
    if free < gib:
        pytest.skip(f"{free:.0f} GiB of device memory free, {gib} needed")


@pytest.fixture(autouse=True)
def _give_back(gpu):
    yield
    torch.cuda.empty_cache()


def _slices(n, launch):
    """Rows at the start, around the end of a launch's rows, and at the end."""
    return [(0, 300), (launch - 300, min(launch + 300, n)), (n - 300, n)]


def test_scales_alone_of_many_splats(gpu):
    """The scales' gradient of a frozen codebook above 2^26 splats."""
    N, K, D = (1 << 26) + 1003, 50, 3
    _room(6)
    g = torch.Generator(device=gpu).manual_seed(1)
    codes = torch.randint(-1, K, (N,), generator=g, device=gpu, dtype=torch.int32)
    book = torch.randn(K, D, generator=g, device=gpu)
    scales = torch.rand(N, generator=g, device=gpu).requires_grad_(True)
    grad = torch.randn(N, D, generator=g, device=gpu)
    got, = torch.autograd.grad(gs.lookup_codes(codes, book, scales, 1.5), scales, grad)
    for a, b in _slices(N, 1 << 26):
        want = R.lookup(codes[a:b].cpu(), book.cpu(), scales[a:b].detach().cpu(), 1.5, grad[a:b].cpu())
        R.check(got[a:b], want["g_scales"], f"rows from {a}")


@pytest.mark.parametrize("N", [0, 1, 3001])
def test_lookup_of_few_splats_in_a_huge_codebook(gpu, N):
    """Every row of the codebook's gradient is written, however few splats there are."""
    K = (1 << 26) + 5
    _room(3)
    book = torch.ones(K, 1, device=gpu, requires_grad=True)
    codes = torch.randint(0, K - 2, (N,), generator=torch.Generator().manual_seed(N)).to(gpu)
    if N:
        codes[0] = K - 2
        codes[N // 2] = K - 2
    junk = torch.full((K, 1), 7.0, device=gpu)  # (what the gradient's memory may hold)
    del junk
    out = gs.lookup_codes(codes, book, None, 3.0)
    g, = torch.autograd.grad(out, book, torch.full((N, 1), 2.0, device=gpu))
    assert out.shape == (N, 1) and bool((out == 3.0).all())
    where, counts = codes.unique(return_counts=True)
    assert torch.equal(g[where, 0], 6.0 * counts)
    assert int(g.count_nonzero()) == where.numel()
