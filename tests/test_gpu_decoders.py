"""Splats' rows by code and back on the GPU: group_codes, rows_by_code and rows_from_codes against the 64-bit
formulas (oracle/decoders_reference.py), whose bounds follow from the roundings of a float32 computation."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _codes(shape, K, seed=0, skew=False, none=0.1, long=False):
    g = _gen(seed)
    codes = torch.randint(0, K, shape, generator=g)
    if skew:
        codes = torch.where(torch.rand(shape, generator=g) < 0.8, torch.full_like(codes, K // 2), codes)
    codes = torch.where(torch.rand(shape, generator=g) < none, torch.full_like(codes, -1), codes)
    return codes if long else codes.to(torch.int32)


def _same_groups(got, want, what=""):
    for name, a, b in zip(("order", "places", "starts"), got, want):
        assert a.dtype == torch.int32 and a.shape == b.shape, f"{what} {name}"
        assert torch.equal(a.cpu(), b), f"{what} {name}: {int((a.cpu() != b).sum())} of {b.numel()} differ"


def _check_group(gpu, codes, K, several=False, what=""):
    got = gs.group_codes(codes.to(gpu), K, several=several)
    want = R.group(codes, K, several)
    _same_groups(got, want, what)
    return got, want


# ---- sorting

SIZES = [1, 2, 63, 64, 65, 255, 256, 257, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8193, 16385, 40000, 65536,
         70001, 300007]


@pytest.mark.parametrize("N", SIZES)
def test_group_sizes(gpu, N):
    for K in (1, 2, 7, 64, 255, 256, 257, 1000, 1024, 4095, 4097, 16384, 70001):
        _check_group(gpu, _codes((N,), K, seed=N + K, skew=K % 2 == 0, long=K % 3 == 0), K, what=f"N={N} K={K}")


@pytest.mark.parametrize("N", [300, 5000, 70001])
@pytest.mark.parametrize("K", [3, 300, 5000])
def test_group_kinds(gpu, N, K):
    """One code alone, none at all, sorted and reversed codes, codes out of range."""
    up = (torch.arange(N) * K // N).to(torch.int32)
    bad = _codes((N,), K, seed=1, long=True)
    bad[::7], bad[3], bad[N // 2] = K, -2, 1 << 40
    for codes in (torch.full((N,), K - 1), torch.zeros(N, dtype=torch.int32), torch.full((N,), -1), up, up.flip(0), bad,
                  torch.where(torch.arange(N) % 2 == 0, -1, K - 1)):
        _check_group(gpu, codes, K, what=f"N={N} K={K}")


def test_group_shapes(gpu):
    c = _codes((3, 5, 4), 9, seed=2)
    assert _check_group(gpu, c, 9)[0].places.shape == (3, 5, 4, 1)
    assert _check_group(gpu, c, 9, several=True)[0].places.shape == (3, 5, 4)
    assert _check_group(gpu, c[0, 0, 0], 9)[0].places.shape == (1,)
    assert _check_group(gpu, c[0, 0], 9, several=True)[0].places.shape == (4,)
    got = gs.group_codes(c.to(gpu).repeat_interleave(2, 1)[:, ::2].transpose(0, 1), 9)
    _same_groups(got, R.group(c.transpose(0, 1), 9))
    for shape in ((0,), (0, 3), (2, 0, 3)):
        for several in (False, len(shape) > 1):
            got = gs.group_codes(torch.zeros(shape, dtype=torch.int64, device=gpu), 5, several=several)
            assert got.order.shape == (0,) and got.starts.tolist() == [0] * 6
            assert got.places.shape == (shape if several else (*shape, 1))


def test_group_huge_codebook(gpu):
    """Many more codes than choices."""
    K = 1 << 24
    codes = torch.tensor([K - 1, 0, 5, -1, K - 1, 12345678], dtype=torch.int32)
    _check_group(gpu, codes, K)
    _check_group(gpu, _codes((9001,), K, seed=4), K)


# ---- rows


def _check_rows(gpu, N, S, K, D, dtype, weights=True, seed=0, skew=False, none=0.1, lead=None, codes=None):
    what = f"N={N} S={S} K={K} D={D} {dtype} weights={weights}"
    g = _gen(seed + 1)
    several = S > 1
    if codes is None:
        codes = _codes((N, S) if several else (N,), K, seed, skew, none)
    shape = lead or (N,)
    codes = codes.reshape(*shape, S) if several else codes.reshape(shape)
    groups, want_groups = _check_group(gpu, codes, K, several, what)
    x = torch.randn(*shape, D, generator=g).to(dtype)
    gy = torch.randn(N * S, D, generator=g).to(dtype)
    want = R.by_code(x, want_groups, gy)
    xg = x.to(gpu).requires_grad_(True)
    y = gs.rows_by_code(xg, groups)
    R.check(y, want["out"], what + " by code")
    R.check(torch.autograd.grad(y, xg, gy.to(gpu))[0], want["g_rows"], what + " by code's gradient")
    rows = torch.randn(N * S, D, generator=g).to(dtype)
    w = torch.randn(codes.shape, generator=g) if weights else None
    go = torch.randn(*shape, D, generator=g).to(dtype)
    want = R.from_codes(rows, want_groups, w, go)
    rg, wg = rows.to(gpu).requires_grad_(True), None if w is None else w.to(gpu).requires_grad_(True)
    out = gs.rows_from_codes(rg, groups, wg)
    R.check(out, want["out"], what + " from codes")
    grads = torch.autograd.grad(out, [rg] + ([wg] if weights else []), go.to(gpu))
    R.check(grads[0], want["g_rows"], what + " g_rows")
    if weights:
        R.check(grads[1], want["g_weights"], what + " g_weights")
    with torch.no_grad():
        assert torch.equal(gs.rows_by_code(xg, groups).nan_to_num(7.0), y.nan_to_num(7.0))
        assert torch.equal(gs.rows_from_codes(rg, groups, wg).nan_to_num(7.0), out.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 7, 8, 9, 11, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 128, 130, 256, 257,
                               512, 520, 1024, 1037, 2050])
def test_rows_widths(gpu, dtype, D):
    _check_rows(gpu, 301, 1, 29, D, dtype, seed=D)
    _check_rows(gpu, 150, 3, 29, D, dtype, weights=D % 2 == 0, seed=D)


@pytest.mark.parametrize("S", [1, 2, 3, 4, 5, 8, 9, 17])
@pytest.mark.parametrize("D,dtype", [(1, F32), (3, F32), (48, BF16), (128, F16), (600, F32)])
def test_rows_choices(gpu, S, D, dtype):
    _check_rows(gpu, 200, S, 13, D, dtype, seed=S)
    _check_rows(gpu, 200, S, 13, D, dtype, weights=False, seed=S)


@pytest.mark.parametrize("N", [1, 2, 63, 64, 65, 1000, 8191, 20011])
@pytest.mark.parametrize("K", [1, 40, 3000])
def test_rows_sizes(gpu, N, K):
    _check_rows(gpu, N, 1, K, 3, F32, seed=N)
    _check_rows(gpu, N, 2, K, 48, BF16, seed=N, skew=True)


@pytest.mark.parametrize("D,dtype", [(3, F32), (64, BF16), (700, F16)])
def test_rows_of_bad_codes(gpu, D, dtype):
    codes = _codes((120, 3), 20, seed=2, long=True)
    codes[5, 0], codes[17, 2], codes[100, 1], codes[119, 2] = 20, -2, 1 << 40, -(1 << 50)
    codes[7], codes[8, 1:] = -1, -1
    _check_rows(gpu, 120, 3, 20, D, dtype, codes=codes)
    _check_rows(gpu, 120, 3, 20, D, dtype, weights=False, codes=codes)
    _check_rows(gpu, 120, 1, 20, D, dtype, codes=codes[:, 0].contiguous())


def test_rows_batch(gpu):
    _check_rows(gpu, 66, 1, 7, 5, F32, lead=(2, 3, 11))
    _check_rows(gpu, 66, 2, 7, 8, BF16, lead=(6, 11))
    _check_rows(gpu, 1, 1, 7, 5, F32, lead=())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [3, 12, 64, 130])
def test_rows_layouts(gpu, dtype, D):
    """Columns of wider rows (at every alignment), every second row, another order of the axes, broadcast rows."""
    N, K, S = 90, 9, 2
    codes = _codes((N, S), K, seed=1)
    groups, want_groups = _check_group(gpu, codes, K, True)
    x, rows = (torch.randn(n, D, generator=_gen(n)).to(dtype) for n in (N, N * S))
    w, go = torch.rand(N, S, generator=_gen(3)), torch.randn(N, D, generator=_gen(4)).to(dtype)
    there, back = R.by_code(x, want_groups)["out"], R.from_codes(rows, want_groups, w, go)

    def views(t):
        for off in (1, 2, 3, 5):
            wide = torch.full((t.shape[0], D + 8), 1e4, dtype=dtype, device=gpu)
            wide[:, off:off + D] = t.to(gpu)
            yield wide[:, off:off + D]
        yield t.to(gpu).repeat_interleave(2, 0)[::2]
        yield t.to(gpu).t().contiguous().t()

    for v in views(x):
        R.check(gs.rows_by_code(v, groups), there, "by code")
    for v in views(rows):
        v = v.detach().requires_grad_(True)
        wg = w.to(gpu).t().contiguous().t().requires_grad_(True)
        out = gs.rows_from_codes(v, groups, wg)
        R.check(out, back["out"], "from codes")
        g = torch.autograd.grad(out, [v, wg], go.to(gpu).t().contiguous().t())
        R.check(g[0], back["g_rows"], "g_rows")
        R.check(g[1], back["g_weights"], "g_weights")
    one = x[:1].expand(N, D)
    R.check(gs.rows_by_code(x[:1].to(gpu).expand(N, D), groups), R.by_code(one, want_groups)["out"], "broadcast")
    y = rows.to(gpu).requires_grad_(True)
    gs.rows_from_codes(y, groups, w.to(gpu)).sum().backward()
    R.check(y.grad, R.from_codes(rows, want_groups, w, torch.ones_like(go))["g_rows"], "gradient of a sum")


def test_rows_one_gradient_at_a_time(gpu):
    codes = _codes((70, 2), 9, seed=5)
    groups, want_groups = _check_group(gpu, codes, 9, True)
    rows, w, go = torch.randn(140, 6, generator=_gen(1)), torch.rand(70, 2, generator=_gen(2)), torch.randn(70, 6, generator=_gen(3))
    want = R.from_codes(rows, want_groups, w, go)
    r = rows.to(gpu).requires_grad_(True)
    R.check(torch.autograd.grad(gs.rows_from_codes(r, groups, w.to(gpu)), r, go.to(gpu))[0], want["g_rows"], "rows alone")
    v = w.to(gpu).requires_grad_(True)
    R.check(torch.autograd.grad(gs.rows_from_codes(rows.to(gpu), groups, v), v, go.to(gpu))[0], want["g_weights"], "weights alone")


def test_rows_empty(gpu):
    for S in (1, 3):
        groups = gs.group_codes(torch.zeros((0, S), dtype=torch.int32, device=gpu), 4, several=True)
        x = torch.zeros(0, 5, device=gpu, requires_grad=True)
        y = gs.rows_by_code(x, groups)
        out = gs.rows_from_codes(y, groups, torch.zeros(0, S, device=gpu, requires_grad=True))
        assert y.shape == (0, 5) and out.shape == (0, 5)
        out.sum().backward()
        assert x.grad.shape == (0, 5)


def test_rows_same_bits(gpu):
    codes = _codes((30000, 3), 60, seed=4, skew=True).to(gpu)
    x, w = torch.randn(30000, 19, device=gpu, requires_grad=True), torch.rand(30000, 3, device=gpu, requires_grad=True)
    first = None
    for _ in range(3):
        groups = gs.group_codes(codes, 60, several=True)
        out = gs.rows_from_codes(gs.rows_by_code(x, groups), groups, w)
        got = [*groups, out, *torch.autograd.grad(out, [x, w], torch.ones_like(out))]
        assert first is None or all(torch.equal(a, b) for a, b in zip(got, first))
        first = got


def test_rows_of_groups_that_are_none(gpu):
    """Places and orders that name no row: NaN or zeros, never an address."""
    x = torch.ones(4, 3, device=gpu)
    i32 = dict(dtype=torch.int32, device=gpu)
    bad = gs.CodeGroups(torch.tensor([0, 7, -5, 1 << 30], **i32), torch.tensor([[0], [9], [-3], [1 << 30]], **i32),
                        torch.tensor([0, 4], **i32))
    y = gs.rows_by_code(x, bad)
    assert bool((y[0] == 1).all()) and bool(y[1:].isnan().all())
    out = gs.rows_from_codes(x, bad)
    assert bool((out[0] == 1).all()) and bool(out[1:].isnan().all())
    w = torch.ones(4, device=gpu, requires_grad=True)
    g = torch.autograd.grad(gs.rows_from_codes(x, bad, w).nan_to_num(0.0).sum(), w)[0]
    assert g.shape == (4,)
