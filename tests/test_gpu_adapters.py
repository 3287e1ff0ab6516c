"""Low-rank maps by code on the GPU: code_adapters against the 64-bit formulas (oracle/decoders_reference.py), whose
bounds follow from the roundings of a float32 computation."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R
from test_gpu_decoders import BF16, F16, F32, _codes, _gen

pytestmark = pytest.mark.gpu


def _inputs(N, K, D, E, r, dtype, seed=0, base=True, skew=False, none=0.1, codes=None):
    g = _gen(seed)
    codes = _codes((N,), K, seed + 1, skew, none) if codes is None else codes
    x, dn, up = torch.randn(N, D, generator=g), torch.randn(K, r, D, generator=g) / D ** 0.5, torch.randn(K, E, r, generator=g)
    b, go = torch.randn(N, E, generator=g), torch.randn(N, E, generator=g)
    return codes, *(t.to(dtype) for t in (x, dn, up)), b.to(dtype) if base else None, go.to(dtype)


def _check(gpu, codes, x, dn, up, b, go, scale=0.75, by_code=False, train=True, what="", several=False):
    K = dn.shape[0]
    what += f" N={x.shape[0]} K={K} D={dn.shape[2]} E={up.shape[1]} r={dn.shape[1]} {x.dtype} by_code={by_code}"
    want = R.adapters(x, R.group(codes, K, several), dn, up, b, scale, by_code, go if train else None)
    groups = gs.group_codes(codes.to(gpu), K, several=several)
    leaves = [None if t is None else t.to(gpu).requires_grad_(train) for t in (x, dn, up, b)]
    out = gs.code_adapters(leaves[0], groups, leaves[1], leaves[2], base=leaves[3], scale=scale, by_code=by_code)
    R.check(out, want["out"], what + " out")
    if not train:
        return
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], go.to(gpu))
    for k, g in zip(("g_rows", "g_down", "g_up"), grads):
        R.check(g, want[k], f"{what} {k}")
    if b is not None:
        assert torch.equal(grads[3].cpu(), go)
    with torch.no_grad():  # (serving: nothing is kept)
        R.check(gs.code_adapters(leaves[0], groups, leaves[1], leaves[2], leaves[3], scale, by_code), want["out"], what + " no grad")


TYPES = [F32, BF16, F16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r", [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128])
def test_ranks(gpu, dtype, r):
    _check(gpu, *_inputs(203, 5, 70, 50, r, dtype, seed=r))
    _check(gpu, *_inputs(37, 9, 128, 96, r, dtype, seed=r, base=False))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 7, 8, 11, 15, 16, 17, 31, 32, 33, 59, 63, 64, 65, 100, 127, 128, 129, 192, 250, 256,
                               257, 500, 512, 520, 1000, 1024, 1030])
def test_widths(gpu, dtype, D):
    _check(gpu, *_inputs(150, 4, D, 40, 8, dtype, seed=D))
    _check(gpu, *_inputs(150, 4, 40, D, 8, dtype, seed=D, base=D % 2 == 0))
    _check(gpu, *_inputs(9, 4, D, D, 16, dtype, seed=D, base=D % 2 == 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 2, 3, 5, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 500, 1000, 2049, 5001])
def test_rows(gpu, dtype, N):
    for K in (1, 3, 40):
        _check(gpu, *_inputs(N, K, 48, 33, 5, dtype, seed=N + K, skew=K == 40))
    _check(gpu, *_inputs(N, 300, 64, 64, 16, dtype, seed=N, none=0.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,D,E,r", [(1, 64, 1024, 1024, 16), (3, 5, 4096, 300, 16), (61, 32, 300, 4096, 16), (7, 7, 4100, 4099, 64),
                                       (700, 40, 1024, 600, 32), (3000, 3, 700, 300, 100), (20, 20, 4096, 4096, 128)])
def test_wide(gpu, dtype, N, K, D, E, r):
    _check(gpu, *_inputs(N, K, D, E, r, dtype, seed=N))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(gpu, dtype):
    """Codes of thousands of rows beside codes of one and of none."""
    codes = torch.cat([torch.full((9000,), 2), torch.tensor([0]), torch.full((4097,), 7), torch.full((64,), 5), torch.full((65,), 6),
                       torch.full((300,), -1)])
    codes = codes[torch.randperm(codes.numel(), generator=_gen(1))]
    for D, E, r in ((40, 24, 12), (130, 70, 33)):
        _check(gpu, *_inputs(codes.numel(), 9, D, E, r, dtype, seed=D, codes=codes))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,E,r", [(100, 24, 31, 4), (700, 130, 64, 32), (5, 600, 1000, 16)])
def test_by_code(gpu, dtype, N, D, E, r):
    _check(gpu, *_inputs(N, 11, D, E, r, dtype, seed=N), by_code=True)
    codes = _codes((N // 5, 5), 11, seed=3)
    _check(gpu, *_inputs(N, 11, D, E, r, dtype, seed=N, codes=codes), by_code=True, several=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("by_code", [False, True])
@pytest.mark.parametrize("N", [40, 1500])
def test_bad_codes(gpu, dtype, by_code, N):
    codes = _codes((N,), 20, seed=2, long=True)
    codes[5], codes[17], codes[30], codes[39] = 20, -2, 1 << 40, -(1 << 50)
    _check(gpu, *_inputs(N, 20, 33, 70, 6, dtype, codes=codes), by_code=by_code)
    _check(gpu, *_inputs(N, 20, 33, 70, 6, dtype, codes=codes, base=False), by_code=by_code)
    _check(gpu, *_inputs(N, 20, 33, 70, 6, dtype, codes=torch.full((N,), -1)), by_code=by_code)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [12, 900])
def test_other_rows_stay_clean(gpu, dtype, N):
    """NaN and infinities in the rows of one code, in the map of one that no splat names, in rows without a code and in
    base there reach nothing else."""
    codes = _codes((N,), 6, seed=1)
    codes[0], codes[1] = 3, -1
    codes = torch.where(codes == 4, torch.full_like(codes, 5), codes)
    codes, x, dn, up, b, go = _inputs(N, 6, 70, 45, 9, dtype, codes=codes)
    want = R.adapters(x, R.group(codes, 6), dn, up, b, 1.0, False, go)
    dn[4], up[4] = float("nan"), float("inf")
    x[codes == -1], x[codes == 3] = float("nan"), float("inf")
    go2 = go.clone()
    go2[codes == -1] = float("inf")
    groups = gs.group_codes(codes.to(gpu), 6)
    leaves = [t.to(gpu).requires_grad_(True) for t in (x, dn, up)]
    out = gs.code_adapters(leaves[0], groups, leaves[1], leaves[2], b.to(gpu))
    grads = torch.autograd.grad(out, leaves, go2.to(gpu))
    clean = codes != 3
    R.check(out[clean.to(gpu)], tuple(t[clean] for t in want["out"]), "out")
    R.check(grads[0][clean.to(gpu)], tuple(t[clean] for t in want["g_rows"]), "g_rows")
    rest = torch.arange(6) != 3
    R.check(grads[1][rest.to(gpu)], tuple(t[rest] for t in want["g_down"]), "g_down")
    R.check(grads[2][rest.to(gpu)], tuple(t[rest] for t in want["g_up"]), "g_up")
    assert not out[~clean.to(gpu)].isfinite().any() and not grads[1][3].isfinite().any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_values(gpu, dtype):
    """Hidden values past the type's range (65504 in float16), results within it."""
    codes, x, dn, up, b, go = _inputs(200, 5, 64, 48, 8, dtype)
    x = (x.float() * 3000).to(dtype)
    dn = (dn.float() * 300).to(dtype)
    up = (up.float() * 2.0 ** -12).to(dtype)
    go = (go.float() * 2.0 ** -8).to(dtype)
    _check(gpu, codes, x, dn, up, b, go, scale=0.25)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,E,r", [(24, 17, 4), (128, 130, 16), (601, 64, 20)])
def test_layouts(gpu, dtype, D, E, r):
    """Columns of wider rows (at every alignment), rows in another order, maps and bases that are views."""
    N, K = 130, 6
    codes, x, dn, up, b, go = _inputs(N, K, D, E, r, dtype)
    want = R.adapters(x, R.group(codes, K), dn, up, b, 0.5, False, go)
    groups = gs.group_codes(codes.to(gpu), K)

    def run(xv, dv, uv, bv, gv):
        leaves = [t.detach().requires_grad_(True) for t in (xv, dv, uv)]
        out = gs.code_adapters(leaves[0], groups, leaves[1], leaves[2], bv, 0.5)
        R.check(out, want["out"], "out")
        for k, g in zip(("g_rows", "g_down", "g_up"), torch.autograd.grad(out, leaves, gv)):
            R.check(g, want[k], k)

    plain = [t.to(gpu) for t in (x, dn, up, b, go)]
    for off in (1, 2, 3, 5):
        wide = torch.full((N, D + 8), 1e4, dtype=dtype, device=gpu)
        wide[:, off:off + D] = plain[0]
        run(wide[:, off:off + D], *plain[1:])
    run(plain[0].t().contiguous().t(), plain[1].transpose(0, 2).contiguous().transpose(0, 2),
        plain[2].transpose(1, 2).contiguous().transpose(1, 2), plain[3].t().contiguous().t(), plain[4].t().contiguous().t())
    # maps that start at any element
    shifted = [torch.cat([t.new_zeros(k + 1), t.reshape(-1)])[k + 1:].view(t.shape) for k, t in enumerate(plain)]
    run(*shifted)
    # a batch
    xb = plain[0].reshape(2, 65, D).requires_grad_(True)
    out = gs.code_adapters(xb, gs.group_codes(codes.to(gpu).reshape(2, 65), K), plain[1], plain[2], plain[3].reshape(2, 65, E), 0.5)
    R.check(out.reshape(N, E), want["out"], "batch")
    R.check(torch.autograd.grad(out, xb, plain[4].reshape(2, 65, E))[0].reshape(N, D), want["g_rows"], "batch g_rows")


@pytest.mark.parametrize("N", [30, 2000])
def test_one_gradient_at_a_time(gpu, N):
    codes, x, dn, up, b, go = _inputs(N, 6, 70, 40, 8, BF16)
    want = R.adapters(x, R.group(codes, 6), dn, up, b, 1.0, False, go)
    groups = gs.group_codes(codes.to(gpu), 6)
    ts = [t.to(gpu) for t in (x, dn, up, b)]
    for k, name in enumerate(("g_rows", "g_down", "g_up")):
        leaf = ts[k].clone().requires_grad_(True)
        args = [leaf if i == k else t for i, t in enumerate(ts)]
        g, = torch.autograd.grad(gs.code_adapters(args[0], groups, *args[1:]), leaf, go.to(gpu))
        R.check(g, want[name], name + " alone")
    leaf = ts[3].clone().requires_grad_(True)
    g, = torch.autograd.grad(gs.code_adapters(ts[0], groups, ts[1], ts[2], leaf), leaf, go.to(gpu))
    assert torch.equal(g.cpu(), go)


def test_empty(gpu):
    dn, up = torch.randn(3, 2, 5, device=gpu, requires_grad=True), torch.randn(3, 4, 2, device=gpu, requires_grad=True)
    for shape in ((0,), (2, 0)):
        groups = gs.group_codes(torch.zeros(shape, dtype=torch.int32, device=gpu), 3)
        out = gs.code_adapters(torch.zeros(*shape, 5, device=gpu), groups, dn, up)
        assert out.shape == (*shape, 4)
        g = torch.autograd.grad(out.sum(), [dn, up])
        assert not g[0].any() and not g[1].any() and g[0].shape == dn.shape and g[1].shape == up.shape


def test_one_row_without_leading_axes(gpu):
    for code in (2, -1):
        codes, x, dn, up, b, go = _inputs(1, 4, 20, 11, 3, F32, codes=torch.tensor([code]))
        want = R.adapters(x, R.group(codes, 4), dn, up, b, 0.5, False, go)
        groups = gs.group_codes(codes[0].to(gpu), 4)
        xg = x[0].to(gpu).requires_grad_(True)
        out = gs.code_adapters(xg, groups, dn.to(gpu), up.to(gpu), b[0].to(gpu), 0.5)
        R.check(out[None], want["out"], "out")
        R.check(torch.autograd.grad(out, xg, go[0].to(gpu))[0][None], want["g_rows"], "g_rows")


def test_rows_that_are_their_own_base(gpu):
    """One tensor in two places: its gradients add up."""
    codes, x, dn, up, _, go = _inputs(300, 5, 32, 32, 8, F32)
    want = R.adapters(x, R.group(codes, 5), dn, up, x, 0.5, False, go)
    xg = x.to(gpu).requires_grad_(True)
    groups = gs.group_codes(codes.to(gpu), 5)
    out = gs.code_adapters(xg, groups, dn.to(gpu), up.to(gpu), xg, 0.5)
    R.check(out, want["out"], "out")
    g, = torch.autograd.grad(out, xg, go.to(gpu))
    value, bound = want["g_rows"]
    total = value + go.double()
    R.check(g, (total, bound + R.E * total.abs() * 2), "g_rows")


def test_same_bits(gpu):
    codes, x, dn, up, b, go = (t.to(gpu) for t in _inputs(20000, 12, 130, 70, 16, BF16, skew=True))
    leaves = [t.requires_grad_(True) for t in (x, dn, up)]
    first = None
    for _ in range(3):
        out = gs.code_adapters(x, gs.group_codes(codes, 12), dn, up, b)
        got = [out, *torch.autograd.grad(out, leaves, go)]
        assert first is None or all(torch.equal(p, q) for p, q in zip(got, first))
        first = got


def test_groups_that_are_none(gpu):
    """Orders and starts that name no row: nothing is read or written past the rows."""
    i32 = dict(dtype=torch.int32, device=gpu)
    x, dn, up = torch.ones(4, 6, device=gpu), torch.ones(2, 3, 6, device=gpu), torch.ones(2, 5, 3, device=gpu)
    for starts in ([0, 2, 4], [0, 9, 4], [-7, 2, 1 << 30], [3, 1, 0], [1 << 30, 1 << 30, 1 << 30]):
        for order in ([0, 7, -5, 1 << 30], [0, 1, 2, 3]):
            bad = gs.CodeGroups(torch.tensor(order, **i32), torch.tensor([[0], [9], [-3], [1 << 30]], **i32), torch.tensor(starts, **i32))
            for by_code in (False, True):
                leaves = [t.clone().requires_grad_(True) for t in (x, dn, up)]
                out = gs.code_adapters(leaves[0], bad, leaves[1], leaves[2], by_code=by_code)
                assert out.shape == (4, 5)
                torch.autograd.grad(out, leaves, torch.ones_like(out))
