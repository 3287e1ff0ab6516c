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


def _rows_check(gpu, N, K, launch, top, train):
    x = torch.empty(N, K, device=gpu, dtype=BF16)
    for a in range(0, N, 1 << 24):
        x[a:a + (1 << 24)].normal_()
    codes = torch.randint(-1, K, (N,), device=gpu, dtype=torch.int32)
    x.requires_grad_(train)
    o = gs.code_log_probs(x, codes, top=top)
    ones = torch.ones(N, device=gpu) if train else None
    g = torch.autograd.grad([o.log_probs, o.entropy], x, [ones, ones])[0] if train else None
    for a, b in _slices(N, launch):
        one = torch.ones(b - a)
        want = R.probs(x[a:b].detach().cpu(), codes[a:b].cpu(), top, 1.0, one if train else None, one if train else None)
        R.check(o.log_probs[a:b], want["log_probs"], f"log_probs from {a}")
        R.check(o.entropy[a:b], want["entropy"], f"entropy from {a}")
        if top:
            R.check(o.top_codes[a:b], want["top_codes"], f"top_codes from {a}")
            R.check(o.top_log_probs[a:b], want["top_log_probs"], f"top_log_probs from {a}")
        if train:
            R.check(g[a:b], want["g_logits"], f"g_logits from {a}")


def test_probs_of_more_rows_than_a_launch_has_wavefronts(gpu):
    """A wavefront a row: 2^26 rows and more."""
    _room(40)
    _rows_check(gpu, (1 << 26) + 1001, 257, 1 << 26, 2, False)


def test_probs_of_more_rows_than_a_launch_has_workgroups(gpu):
    """A workgroup a row: 2^24 rows and more."""
    _room(75)
    _rows_check(gpu, (1 << 24) + 1001, 2056, 1 << 24, 1, False)


def test_probs_gradient_of_more_rows_than_a_launch_has_teams(gpu):
    """Eight lanes a row: 2^29 rows and more."""
    _room(110)
    _rows_check(gpu, (1 << 29) + 1001, 33, 1 << 29, 0, True)


def test_sizes_past_32_bits_are_refused(gpu):
    """On the host path too: one value broadcast to more than 2^32."""
    past = (1 << 32) + 7
    one, code = torch.zeros(1, 1, device=gpu, dtype=BF16), torch.zeros(1, device=gpu, dtype=torch.int32)
    for f in (lambda x: gs.lookup_codes(code, x.expand(past, 1)), lambda x: gs.lookup_codes(code, x.expand(1, past)),
              lambda x: gs.code_log_probs(x.expand(1, past), code), lambda x: gs.code_balance(x.expand(1, past), code),
              lambda x: gs.code_balance(x[None].expand(past, 1, 1), code[None].expand(past, 1)),
              lambda x: gs.code_balance(x, code[None].expand(1, past))):
        for train in (False, True):
            with pytest.raises(ValueError, match=r"are supported, not 4294967303"):
                f(one.clone().requires_grad_(train))
