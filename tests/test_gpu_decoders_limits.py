"""Decoders by code and clipping at sizes past one launch's threads, past 32 bits, and past one way of sorting."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _room(gib):
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0] / 2 ** 30
    if free < gib:
        pytest.skip(f"{free:.0f} GiB of device memory free, {gib} needed")


@pytest.fixture(autouse=True)
def _give_back(gpu):
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("N,K", [((1 << 22) + 77, 100), ((1 << 22) - 5, 2047), (3000001, 5000), (1 << 25, 60), ((1 << 25) + 9, 60)])
def test_sort(gpu, N, K):
    codes = torch.randint(-1, K, (N,), device=gpu, dtype=torch.int32)
    got = gs.group_codes(codes, K)
    keys = torch.where(codes >= 0, codes, K).long()
    order = torch.sort(keys, stable=True).indices
    assert torch.equal(got.order.long(), order)
    places = torch.empty_like(order)
    places[order] = torch.arange(N, device=gpu)
    assert torch.equal(got.places[:, 0].long(), torch.where(codes >= 0, places, -1))
    assert torch.equal(got.starts.long(), torch.searchsorted(keys[order], torch.arange(K + 1, device=gpu)))


def test_adapters_of_more_tiles_than_a_launch_has_workgroups(gpu):
    """2^29 rows, more than 2^32 values in and out."""
    _room(60)
    N, K, D, E, r = 1 << 29, 3, 9, 10, 100
    x = torch.empty(N, D, device=gpu, dtype=BF16)
    for a in range(0, N, 1 << 26):
        x[a:a + (1 << 26)].normal_()
    codes = torch.randint(-1, K, (N,), device=gpu, dtype=torch.int32)
    dn, up = torch.randn(K, r, D, device=gpu).to(BF16), torch.randn(K, E, r, device=gpu).to(BF16)
    groups = gs.group_codes(codes, K)
    out = gs.code_adapters(x, groups, dn, up)
    del groups
    for a in (0, N // 3, N - 500):
        part = codes[a:a + 500].cpu()
        want = R.adapters(x[a:a + 500].cpu(), R.group(part, K), dn.cpu(), up.cpu())
        R.check(out[a:a + 500], want["out"], f"rows from {a}")


@pytest.mark.parametrize("N", [0, 5, 3000])
def test_adapters_of_more_codes_than_a_launch_has_workgroups(gpu, N):
    """Every map's gradient is written, however few rows there are."""
    _room(4)
    K = (1 << 24) + 3
    codes = torch.randint(0, K - 2, (N,), generator=torch.Generator().manual_seed(N)).to(gpu)
    if N:
        codes[0], codes[N // 2] = K - 2, K - 2
    dn, up = torch.full((K, 1, 2), 2.0, device=gpu, requires_grad=True), torch.full((K, 3, 1), 3.0, device=gpu, requires_grad=True)
    junk = torch.full((K, 3), 7.0, device=gpu)  # (what the gradients' memory may hold)
    del junk
    x = torch.ones(N, 2, device=gpu)
    out = gs.code_adapters(x, gs.group_codes(codes, K), dn, up)
    assert out.shape == (N, 3) and bool((out == 12.0).all())
    g_down, g_up = torch.autograd.grad(out, [dn, up], torch.ones_like(out))
    where, counts = codes.unique(return_counts=True)
    assert torch.equal(g_down[where], (9.0 * counts)[:, None, None].expand(-1, 1, 2))
    assert torch.equal(g_up[where], (4.0 * counts)[:, None, None].expand(-1, 3, 1))
    assert int(g_down.count_nonzero()) == 2 * where.numel() and int(g_up.count_nonzero()) == 3 * where.numel()


def test_adapters_gradient_past_32_bits(gpu):
    """More than 2^32 values of rows and results, one code of most rows: chunks by the thousand."""
    _room(120)
    N, K, D, E, r = (1 << 24) + 5, 3, 260, 264, 4
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.empty(N, D, device=gpu, dtype=BF16)
    for a in range(0, N, 1 << 22):
        x[a:a + (1 << 22)] = torch.randint(-2, 3, (min(1 << 22, N - a), D), device=gpu, generator=g).to(BF16)
    codes = torch.where(torch.rand(N, device=gpu, generator=g) < 0.9, 1, 2).to(torch.int32)
    dn = torch.randint(-1, 2, (K, r, D), device=gpu, generator=g).to(BF16).requires_grad_(True)
    up = torch.randint(-1, 2, (K, E, r), device=gpu, generator=g).to(BF16).requires_grad_(True)
    x.requires_grad_(True)
    out = gs.code_adapters(x, gs.group_codes(codes, K), dn, up)
    one = torch.ones((), device=gpu, dtype=BF16).expand(N, E).contiguous()
    gx, g_down, g_up = torch.autograd.grad(out, [x, dn, up], one)
    # g = 1: dh = the columns' sums of up, whole numbers; gdown[c] = dh sum x, gup[c] = sum h: whole numbers below 2^24
    # a chunk, so that only the chunks' sums and the last rounding are off
    dh = up.detach().double().sum(1)
    for c in range(K):
        total = torch.zeros(D, dtype=torch.float64, device=gpu)
        size = 0
        for a in range(0, N, 1 << 20):
            rows = x.detach()[a:a + (1 << 20)][codes[a:a + (1 << 20)] == c]
            total += rows.double().sum(0)
            size += rows.shape[0]
        want = dh[c][:, None] * total
        bound = 2.0 ** -8 * want.abs() + R.E * 2048 * 2 * size * dh[c].abs()[:, None] + 1e-30
        assert bool(((g_down[c].double() - want).abs() <= bound).all()), c
        h = dn.detach()[c].double() @ total
        want = h.expand(E, r)
        bound = 2.0 ** -8 * want.abs() + R.E * 2048 * 2 * size * D + 1e-30
        assert bool(((g_up[c].double() - want).abs() <= bound).all()), c
    for a in (0, N // 2, N - 300):
        c = codes[a:a + 300].long()
        want = torch.matmul(dh[c].unsqueeze(1), dn.detach().double()[c]).squeeze(1)
        assert torch.equal(gx[a:a + 300].double(), want.to(BF16).double())


def test_rows_past_32_bits(gpu):
    _room(60)
    N, D, K = (1 << 23) + 11, 520, 40
    codes = torch.randint(-1, K, (N,), device=gpu, dtype=torch.int32)
    groups = gs.group_codes(codes, K)
    x = torch.empty(N, D, device=gpu, dtype=BF16)
    for a in range(0, N, 1 << 21):
        x[a:a + (1 << 21)].normal_()
    y = gs.rows_by_code(x, groups)
    named = int(groups.starts[-1])
    for a in (0, named // 2, named - 700):
        assert torch.equal(y[a:a + 700], x[groups.order[a:a + 700].long()])
    assert not y[named:].any()
    back = gs.rows_from_codes(y, groups)
    for a in (0, N // 2, N - 700):
        assert torch.equal(back[a:a + 700], torch.where(codes[a:a + 700, None] >= 0, x[a:a + 700], 0))


def test_clip_past_32_bits(gpu):
    _room(30)
    n = (1 << 32) + 12345
    t = torch.full((n,), 0.5, device=gpu, dtype=BF16)
    more = torch.full((10,), 0.5, device=gpu)
    norm = gs.clip_gradients([t, more], 2.0 ** 14)
    want = 0.5 * (n + 10) ** 0.5
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    value = torch.tensor(0.5 * 2.0 ** 14 / want).to(BF16)
    assert bool((t[:: (1 << 20) + 1] == value.to(gpu)).all()) and bool((t[-5:] == value.to(gpu)).all())
