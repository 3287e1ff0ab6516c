"""Scenes in codes on the GPU: lookup_codes, code_log_probs and code_balance against the 64-bit
formulas (oracle/codes_reference.py), whose bounds follow from the roundings of a float32 computation."""
import math

import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import codes_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- lookup


def _lookup_inputs(shape, K, D, dtype, long=False, scales=True, skew=False, seed=0):
    g = _gen(seed)
    codes = torch.randint(0, K, shape, generator=g)
    if skew:
        codes = torch.where(torch.rand(shape, generator=g) < 0.8, torch.full_like(codes, K // 2), codes)
    codes = torch.where(torch.rand(shape, generator=g) < 0.1, torch.full_like(codes, -1), codes)
    codes = codes if long else codes.to(torch.int32)
    book = torch.randn(K, D, generator=g).to(dtype)
    s = torch.randn(shape, generator=g).exp() if scales else None
    grad = torch.randn(*shape, D, generator=g).to(dtype)
    return codes, book, s, grad


def _check_lookup(gpu, codes, book, s, grad, factor=1.0, what=""):
    want = R.lookup(codes, book, s, factor, grad)
    b = book.to(gpu).requires_grad_(True)
    sg = None if s is None else s.to(gpu).requires_grad_(True)
    out = gs.lookup_codes(codes.to(gpu), b, sg, factor)
    R.check(out, want["out"], what + " out")
    grads = torch.autograd.grad(out, [b] + ([] if s is None else [sg]), grad.to(gpu))
    R.check(grads[0], want["g_codebook"], what + " g_codebook")
    if s is not None:
        R.check(grads[1], want["g_scales"], what + " g_scales")
    with torch.no_grad():
        assert torch.equal(gs.lookup_codes(codes.to(gpu), b, sg, factor).nan_to_num(7.0), out.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [1, 2, 3, 4, 8, 11, 17, 48, 63, 64, 65, 130, 256, 520, 1037])
def test_lookup_widths(gpu, dtype, D):
    _check_lookup(gpu, *_lookup_inputs((403,), 29, D, dtype, seed=D), what=f"D={D} {dtype}")


@pytest.mark.parametrize("N", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 4096, 4097, 9001])
@pytest.mark.parametrize("K", [1, 2, 255, 256, 257, 5000])
def test_lookup_sizes(gpu, N, K):
    _check_lookup(gpu, *_lookup_inputs((N,), K, 3, F32, long=N % 2 == 0, scales=K % 2 == 0, skew=N > 128, seed=N + K),
                  factor=1.5, what=f"N={N} K={K}")


@pytest.mark.parametrize("D,dtype", [(3, F32), (11, BF16), (48, F16), (128, F32)])
def test_lookup_runs_over_many_pieces(gpu, D, dtype):
    """One code of most splats, beside codes of few or no splats; and the largest sort."""
    _check_lookup(gpu, *_lookup_inputs((20011,), 300, D, dtype, skew=True, seed=D), what=f"D={D}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64, 65, 100, 130, 256, 257, 512, 520, 1037])
def test_lookup_widths_of_many_splats(gpu, dtype, D):
    """Above the splats that one launch takes: runs of one to hundreds of splats, rows of every team's width."""
    _check_lookup(gpu, *_lookup_inputs((8200 + D,), 2000, D, dtype, skew=D % 2 == 0, seed=D), what=f"D={D} {dtype}")


@pytest.mark.parametrize("N", [8193, 8200, 16384, 65536, 70001, 262145])
def test_lookup_run_ends(gpu, N):
    """Runs that end at, before and after the cuts of the sorted positions; one run of all; one run each."""
    g = _gen(N)
    K = 40000
    for codes in (torch.arange(N) // 64 % K, torch.arange(N) // 63 % K, torch.zeros(N, dtype=torch.long) + 7,
                  torch.arange(N) // 1024, torch.full((N,), -1), torch.arange(N) % K,
                  torch.cat([torch.full((N // 2,), -1), torch.full((N - N // 2,), K - 1)])):
        codes = codes[torch.randperm(N, generator=g)].to(torch.int32)
        for D, scales in ((3, True), (24, False)):
            _check_lookup(gpu, codes, torch.randn(K, D, generator=g), torch.rand(N, generator=g) if scales else None,
                          torch.randn(N, D, generator=g), what=f"N={N} D={D}")


@pytest.mark.parametrize("K", [70001, 1 << 18])
def test_lookup_large_codebook(gpu, K):
    codes, book, s, grad = _lookup_inputs((6007,), K, 4, F32, seed=3)
    codes[0], codes[1] = K - 1, 0
    _check_lookup(gpu, codes, book, s, grad, what=f"K={K}")


def test_lookup_batch_and_odd_layouts(gpu):
    codes, book, s, grad = _lookup_inputs((3, 211), 40, 5, F32, seed=1)
    want = R.lookup(codes, book, s, 1.0, grad)
    # columns of a wider codebook, codes and scales of every second splat, a gradient in another order
    wide = torch.randn(40, 13, device=gpu)
    wide[:, 3:8] = book.to(gpu)
    c2 = codes.to(gpu).repeat_interleave(2, dim=1)[:, ::2]
    s2 = s.to(gpu).t().contiguous().t().requires_grad_(True)
    wide.requires_grad_(True)
    out = gs.lookup_codes(c2, wide[:, 3:8], s2)
    R.check(out, want["out"], "out")
    g2 = grad.to(gpu).permute(2, 1, 0).contiguous().permute(2, 1, 0)
    gw, g_s = torch.autograd.grad(out, [wide, s2], g2)
    R.check(gw[:, 3:8], want["g_codebook"], "g_codebook")
    assert not gw[:, :3].any() and not gw[:, 8:].any()
    R.check(g_s, want["g_scales"], "g_scales")
    # a codebook whose columns are the strided axis, and a gradient that is broadcast
    t = book.to(gpu).t().contiguous().t().requires_grad_(True)
    out = gs.lookup_codes(codes.to(gpu), t)
    R.check(out, R.lookup(codes, book)["out"], "out of a transposed codebook")
    out.sum().backward()
    R.check(t.grad, R.lookup(codes, book, None, 1.0, torch.ones_like(grad))["g_codebook"], "g of a sum")


def test_lookup_bad_codes_and_empty(gpu):
    codes, book, s, grad = _lookup_inputs((300,), 20, 6, F32, long=True, seed=2)
    codes[5], codes[17], codes[100], codes[299] = 20, -2, 1 << 40, -(1 << 50)
    _check_lookup(gpu, codes, book, s, grad, what="bad codes")
    for shape in ((0,), (2, 0)):
        b = torch.randn(7, 3, device=gpu, requires_grad=True)
        out = gs.lookup_codes(torch.zeros(shape, dtype=torch.int32, device=gpu), b)
        assert out.shape == (*shape, 3)
        out.sum().backward()
        assert b.grad.shape == (7, 3) and not b.grad.any()
    b = torch.randn(7, 3, device=gpu, requires_grad=True)
    gs.lookup_codes(torch.full((50,), -1, device=gpu), b).sum().backward()
    assert not b.grad.any()


def test_lookup_same_bits(gpu):
    codes, book, s, grad = (t.to(gpu) for t in _lookup_inputs((30000,), 60, 19, F32, skew=True, seed=4))
    book.requires_grad_(True)
    first = None
    for _ in range(4):
        g, = torch.autograd.grad(gs.lookup_codes(codes, book, s), book, grad)
        assert first is None or torch.equal(g, first)
        first = g


def test_lookup_one_gradient_at_a_time(gpu):
    codes, book, s, grad = (t.to(gpu) for t in _lookup_inputs((700,), 60, 9, F32, seed=5))
    want = R.lookup(codes.cpu(), book.cpu(), s.cpu(), 1.0, grad.cpu())
    b = book.clone().requires_grad_(True)
    R.check(torch.autograd.grad(gs.lookup_codes(codes, b, s), b, grad)[0], want["g_codebook"], "codebook alone")
    s1 = s.clone().requires_grad_(True)
    R.check(torch.autograd.grad(gs.lookup_codes(codes, book, s1), s1, grad)[0], want["g_scales"], "scales alone")


def test_lookup_past_32_bits(gpu):
    """Outputs of more than 2^32 values: the last splats get what a call of them alone gives."""
    N, D = (1 << 23) + 5, 520
    book = torch.randn(64, D, device=gpu).to(BF16)
    codes = torch.randint(0, 64, (N,), device=gpu, dtype=torch.int32)
    out = gs.lookup_codes(codes, book)
    for a, b in ((0, 1000), (N // 2, N // 2 + 1000), (N - 1000, N)):
        assert torch.equal(out[a:b], gs.lookup_codes(codes[a:b], book))
    del out
    book.requires_grad_(True)
    out = gs.lookup_codes(codes, book)
    g, = torch.autograd.grad(out, book, torch.ones((), device=gpu, dtype=BF16).expand_as(out).contiguous())
    counts = torch.bincount(codes, minlength=64)
    assert torch.equal(g, counts.float()[:, None].expand(64, D).to(BF16))  # (counts below 2^24: sums are exact)


# ---- log probabilities


def _logits(shape, K, dtype, seed=0, masked=0.0, spread=3.0):
    g = _gen(seed)
    x = spread * torch.randn(*shape, K, generator=g)
    if masked:
        x[torch.rand(*shape, K, generator=g) < masked] = -math.inf
    return x.to(dtype)


def _check_probs(gpu, x, codes, top, T=1.0, train=True, what="", view=None, seed=9):
    g = _gen(seed)
    shape = x.shape[:-1]
    gl = torch.randn(shape, generator=g) if codes is not None else None
    ge, gt = torch.randn(shape, generator=g), (torch.randn(*shape, top, generator=g) if top else None)
    want = R.probs(x, codes, top, T, gl, ge, gt)
    xg = (view(x) if view else x.to(gpu)).requires_grad_(train)
    cg = None if codes is None else codes.to(gpu)
    o = gs.code_log_probs(xg, cg, top=top, temperature=T)
    if codes is None:
        assert o.log_probs is None
    else:
        R.check(o.log_probs, want["log_probs"], what + " log_probs")
    R.check(o.entropy, want["entropy"], what + " entropy")
    if top:
        R.check(o.top_codes, want["top_codes"], what + " top_codes")
        R.check(o.top_log_probs, want["top_log_probs"], what + " top_log_probs")
    else:
        assert o.top_codes is None and o.top_log_probs is None
    if train:
        outs = [(o.log_probs, gl), (o.entropy, ge), (o.top_log_probs, gt)]
        outs = [(a, b.to(gpu)) for a, b in outs if a is not None]
        got, = torch.autograd.grad([a for a, _ in outs], xg, [b for _, b in outs])
        R.check(got, want["g_logits"], what + " g_logits")
    return o


KS = [1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 500, 512, 513, 1000, 1023,
      1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193]


@pytest.mark.parametrize("K", KS)
def test_probs_codes(gpu, K):
    for dtype, rows, top in ((F32, 5, min(K, 4)), (BF16, 70, min(K, 1)), (F16, 3, 0)):
        x = _logits((rows,), K, dtype, seed=K, masked=0.1 if K > 2 else 0.0)
        codes = torch.randint(-1, K, (rows,), generator=_gen(K + 1))
        _check_probs(gpu, x, codes, top, what=f"K={K} {dtype}")


@pytest.mark.parametrize("K", [16383, 16384, 16385, 20000, 32768, 32771, 65536, 131072, 200003])
@pytest.mark.parametrize("rows", [1, 3])
def test_probs_long_rows(gpu, K, rows):
    dtype = F32 if rows == 1 else BF16
    x = _logits((rows,), K, dtype, seed=K)
    codes = torch.randint(0, K, (rows,), generator=_gen(K + 1)).to(torch.int32)
    _check_probs(gpu, x, codes, 8, T=0.7, what=f"K={K} rows={rows}")


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 63, 64, 65, 1000, 4001])
@pytest.mark.parametrize("K,top", [(8, 2), (40, 1), (257, 20)])
def test_probs_rows(gpu, rows, K, top):
    x = _logits((rows,), K, F32, seed=rows)
    _check_probs(gpu, x, torch.randint(-1, K, (rows,), generator=_gen(rows)), top, T=2.0, what=f"rows={rows} K={K}")


@pytest.mark.parametrize("top", [1, 2, 5, 16, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("K", [64, 200, 3000, 40000])
def test_probs_top(gpu, top, K):
    _check_probs(gpu, _logits((6,), K, F32, seed=top), None, top, train=K < 40000, what=f"top={top} K={K}")


@pytest.mark.parametrize("K", [5, 64, 300, 2500, 9000, 33000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_probs_ties(gpu, K, dtype):
    """Equal logits: the lower codes first, among -0 and +0 too."""
    top = min(K, 12)
    x = torch.zeros(6, K)
    x[1] = -3.5
    x[2, K // 2:] = 1.0
    x[3, ::2] = -0.0
    x[4] = torch.randint(0, 3, (K,), generator=_gen(K)).float()
    x[5] = torch.arange(K).flip(0).div(4, rounding_mode="floor").float().clamp(max=200)
    _check_probs(gpu, x.to(dtype), torch.arange(6) % K, top, what=f"ties K={K}")
    rising = torch.linspace(-5, 5, K).expand(2, K).contiguous()
    rising[1] = rising[0].flip(0)
    _check_probs(gpu, rising.to(dtype), None, top, what=f"ordered K={K}")


@pytest.mark.parametrize("K", [6, 64, 257, 2000, 9001, 40000])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_probs_masks(gpu, K, dtype):
    """Rows with nothing, with one code, with the type's lowest value, with infinities and NaN."""
    x = _logits((10,), K, dtype, seed=K)
    low = torch.finfo(dtype).min
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, K // 2] = 0.25
    x[2] = low
    x[3] = low
    x[3, 1] = 2.0
    x[4, : K // 2] = low
    x[5, K - 1] = math.inf
    x[6, K // 3] = math.nan
    x[7] = -math.inf
    x[7, 2] = math.nan
    x[8, 1::2] = -math.inf
    x[9] = torch.finfo(dtype).max
    codes = torch.tensor([1, K // 2, 0, 0, K - 1, 2, 0, -1, 1, 3])
    # one alternative more than the second row has codes: the masked ones follow in their order
    _check_probs(gpu, x, codes, 3, what=f"masks K={K}")
    _check_probs(gpu, x, codes, 3, T=0.25, what=f"masks K={K} T=0.25")


def test_probs_bad_codes_and_empty(gpu):
    x = _logits((40,), 33, F32, seed=1)
    codes = torch.randint(0, 33, (40,), generator=_gen(2))
    codes[3], codes[7], codes[11] = 33, -2, 1 << 35
    _check_probs(gpu, x, codes, 2, what="bad codes")
    x0 = torch.empty(2, 0, 9, device=gpu, requires_grad=True)
    o = gs.code_log_probs(x0, torch.empty(2, 0, dtype=torch.int32, device=gpu), top=2)
    assert o.log_probs.shape == (2, 0) and o.top_codes.shape == (2, 0, 2)
    o.entropy.sum().backward()
    assert x0.grad.shape == x0.shape
    # one row without any leading axis
    x1 = _logits((1,), 50, F32, seed=3)[0]
    _check_probs(gpu, x1, torch.tensor(7), 3, what="no leading axis")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("K", [13, 130, 1027, 8200])
def test_probs_layouts(gpu, dtype, K):
    """Columns of wider logits (rows at every alignment), every second row, rows in another order."""
    x = _logits((9,), K, dtype, seed=K)
    codes = torch.randint(-1, K, (9,), generator=_gen(4))
    for off in (1, 2, 3, 5):
        def columns(x):
            wide = torch.full((9, K + 8), 1e4, dtype=dtype, device=gpu)
            wide[:, off:off + K] = x.to(gpu)
            return wide[:, off:off + K].detach()
        _check_probs(gpu, x, codes, 2, what=f"columns from {off}", view=columns)
    _check_probs(gpu, x, codes, 2, what="second rows", view=lambda x: x.to(gpu).repeat_interleave(2, 0)[::2].detach())
    _check_probs(gpu, x, codes, 2, what="transposed", view=lambda x: x.to(gpu).t().contiguous().t().detach())
    row = x[:1].expand(9, K)
    _check_probs(gpu, row, codes, 2, what="broadcast", view=lambda x: x[:1].to(gpu).expand(9, K).detach())
    b = x.reshape(3, 3, K)
    _check_probs(gpu, b, codes.reshape(3, 3), 2, what="batch order",
                 view=lambda x: x.to(gpu).transpose(0, 1).contiguous().transpose(0, 1).detach())


def test_probs_gradients_one_at_a_time(gpu):
    x = _logits((50,), 90, F32, seed=5)
    codes = torch.randint(0, 90, (50,), generator=_gen(6))
    g = torch.randn(50, generator=_gen(7))
    gt = torch.randn(50, 3, generator=_gen(8))
    for kw, pick in ((dict(g_log_probs=g), "log_probs"), (dict(g_entropy=g), "entropy"), (dict(g_top=gt), "top_log_probs")):
        xg = x.to(gpu).requires_grad_(True)
        o = gs.code_log_probs(xg, codes.to(gpu), top=3)
        got, = torch.autograd.grad(getattr(o, pick), xg, next(iter(kw.values())).to(gpu))
        R.check(got, R.probs(x, codes, 3, 1.0, **kw)["g_logits"], pick)


def test_probs_past_32_bits(gpu):
    N, K = (1 << 20) + 3, 2051
    x = torch.randn(N, K, device=gpu, dtype=torch.bfloat16)
    codes = torch.randint(0, K, (N,), device=gpu)
    x.requires_grad_(True)
    o = gs.code_log_probs(x, codes, top=2)
    g, = torch.autograd.grad([o.log_probs, o.entropy], x, [torch.ones(N, device=gpu), torch.ones(N, device=gpu)])
    bal = gs.code_balance(x, codes)
    for a, b in ((0, 64), (N - 64, N)):
        part = x[a:b].detach().clone().requires_grad_(True)
        p = gs.code_log_probs(part, codes[a:b], top=2)
        ones = torch.ones(b - a, device=gpu)
        gp, = torch.autograd.grad([p.log_probs, p.entropy], part, [ones, ones])
        assert torch.equal(o.top_codes[a:b], p.top_codes)
        for u, v, w in ((o.log_probs[a:b], p.log_probs, 1e-5), (o.entropy[a:b], p.entropy, 1e-5), (g[a:b].float(), gp.float(), 2.0 ** -7)):
            assert float((u - v).abs().max()) <= w * float(v.abs().max())
    assert int(bal.counts.sum()) == N and torch.equal(bal.counts, torch.bincount(codes, minlength=K).to(torch.int32))
    assert abs(float(bal.mean_probs.double().sum()) - 1.0) < 1e-4


# ---- balance


def _check_balance(gpu, x, codes, train=True, what="", view=None, seed=11):
    g = _gen(seed)
    gl = torch.randn(x.shape[:-2], generator=g)
    gm = torch.randn(*x.shape[:-2], x.shape[-1], generator=g)
    if x.dtype == F16:  # (gradients in 16 bits: a scaled loss)
        gl, gm = gl * x.shape[-2], gm * x.shape[-2]
    want = R.balance(x, codes, gl, gm)
    xg = (view(x) if view else x.to(gpu)).requires_grad_(train)
    o = gs.code_balance(xg, codes.to(gpu))
    for k in ("counts", "mean_probs", "loss"):
        R.check(getattr(o, k), want[k], f"{what} {k}")
    if train:
        got, = torch.autograd.grad([o.loss, o.mean_probs], xg, [gl.to(gpu), gm.to(gpu)])
        R.check(got, want["g_logits"], what + " g_logits")
    return o


@pytest.mark.parametrize("K", [1, 2, 3, 8, 13, 32, 33, 64, 65, 127, 128, 130, 256, 257, 512, 1000, 1024, 1025, 2048, 2050, 4096,
                               4097, 8192, 8200, 16384, 16390, 33000, 70000])
def test_balance_codes(gpu, K):
    for dtype, rows in ((F32, 37), (BF16, 70), (F16, 5)):
        if K > 5000:
            rows = 6
        x = _logits((rows,), K, dtype, seed=K, masked=0.1 if K > 2 else 0.0)
        codes = torch.randint(-1, K, (rows,), generator=_gen(K))
        _check_balance(gpu, x, codes, what=f"K={K} {dtype}")


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 5003])
@pytest.mark.parametrize("K", [8, 50, 300])
def test_balance_rows(gpu, rows, K):
    x = _logits((rows,), K, F32, seed=rows)
    _check_balance(gpu, x, torch.randint(-1, K, (rows,), generator=_gen(rows)).to(torch.int32), what=f"rows={rows} K={K}")


@pytest.mark.parametrize("B,G,K,S", [(2, 100, 20, 2), (5, 33, 130, 4), (3, 1, 7, 3), (7, 1030, 66, 1), (2, 40, 3000, 2)])
def test_balance_batches_and_choices(gpu, B, G, K, S):
    x = _logits((B, G), K, F32, seed=G, masked=0.2)
    codes = torch.randint(-1, K, (B, G, S), generator=_gen(G))
    codes[0, : G // 2] = -1                                      # rows that take no part
    codes[1][torch.rand(G, S, generator=_gen(1)) < 0.8] = K // 2  # a hot code
    x[B - 1, :] = -math.inf                                       # an image whose rows have no logit
    if B > 2:
        codes[2] = -1                                             # an image without any code
    o = _check_balance(gpu, x, codes, what=f"B={B} G={G} K={K} S={S}")
    if B > 2:
        assert float(o.loss[2].detach()) == 0.0


def test_balance_masks_nan_and_bad_codes(gpu):
    x = _logits((4, 20), 30, F32, seed=2)
    codes = torch.randint(0, 30, (4, 20), generator=_gen(3))
    codes[0, 4] = 30
    codes[1, 5] = -2
    x[2, 3, 7] = math.nan
    x[2, 4] = torch.finfo(F32).min
    x[3, 5] = -math.inf
    x[3, 6] = torch.finfo(F32).max
    codes[3, 7] = -1
    x[3, 7] = math.nan  # (in a row that takes no part)
    want = R.balance(x, codes)
    o = gs.code_balance(x.to(gpu), codes.to(gpu))
    for k in ("counts", "mean_probs", "loss"):
        R.check(getattr(o, k), want[k], k)


@pytest.mark.parametrize("K", [30, 700, 3001, 20000])
def test_balance_gradient_of_rows_without_part(gpu, K):
    """NaN and infinities in rows without a code reach nothing; a NaN in a row with one makes its row NaN."""
    for dtype in (F32, BF16):
        x = _logits((9,), K, dtype, seed=K)
        codes = torch.randint(0, K, (9,), generator=_gen(K))
        codes[2] = codes[3] = codes[4] = -1
        x[2, 1] = math.nan
        x[3, 2] = math.inf
        x[4] = -math.inf
        x[5] = -math.inf
        _check_balance(gpu, x, codes, what=f"no part K={K} {dtype}")
        g_loss = torch.ones(())
        x[6, 3] = math.nan
        want = R.balance(x, codes, g_loss, torch.zeros(K))["g_logits"]
        xg = x.to(gpu).requires_grad_(True)
        o = gs.code_balance(xg, codes.to(gpu))
        got, = torch.autograd.grad(o.loss, xg, torch.ones((), device=gpu))
        R.check(got, want, f"NaN row K={K} {dtype}")


@pytest.mark.parametrize("N", [700, 9000])
def test_lookup_gradients_of_splats_without_code(gpu, N):
    """NaN and infinities in the gradient of splats without a code reach no row of the codebook."""
    codes, book, s, grad = _lookup_inputs((N,), 50, 12, F32, seed=N)
    none = codes < 0
    clean = grad.clone()
    clean[none] = 0.0
    grad[none] = math.nan
    grad[none.nonzero()[0]] = math.inf
    want = R.lookup(codes, book, s, 1.0, clean)
    b, sg = book.to(gpu).requires_grad_(True), s.to(gpu).requires_grad_(True)
    gb, g_s = torch.autograd.grad(gs.lookup_codes(codes.to(gpu), b, sg), [b, sg], grad.to(gpu))
    R.check(gb, want["g_codebook"], "g_codebook")
    R.check(g_s, want["g_scales"], "g_scales")


def test_balance_layouts_and_empty(gpu):
    x = _logits((2, 60), 19, F32, seed=4)
    codes = torch.randint(-1, 19, (2, 60), generator=_gen(5))

    def columns(x):
        wide = torch.zeros(2, 60, 30, device=gpu)
        wide[..., 7:26] = x.to(gpu)
        return wide[..., 7:26].detach()
    _check_balance(gpu, x, codes, what="columns", view=columns)
    _check_balance(gpu, x, codes, what="batch order", view=lambda x: x.to(gpu).transpose(0, 1).contiguous().transpose(0, 1).detach())
    x0 = torch.empty(2, 0, 9, device=gpu, requires_grad=True)
    o = gs.code_balance(x0, torch.empty(2, 0, dtype=torch.int32, device=gpu))
    assert not o.loss.any() and not o.counts.any() and not o.mean_probs.any()
    o.loss.sum().backward()
    assert x0.grad.shape == x0.shape


def test_balance_gradients_one_at_a_time(gpu):
    x = _logits((90,), 40, F32, seed=6)
    codes = torch.randint(0, 40, (90,), generator=_gen(7))
    gm = torch.randn(40, generator=_gen(8))
    xg = x.to(gpu).requires_grad_(True)
    o = gs.code_balance(xg, codes.to(gpu))
    one = torch.ones(())
    R.check(torch.autograd.grad(o.loss, xg, retain_graph=True)[0], R.balance(x, codes, one)["g_logits"], "loss")
    R.check(torch.autograd.grad(o.mean_probs, xg, gm.to(gpu))[0], R.balance(x, codes, None, gm)["g_logits"], "mean")


def test_same_bits(gpu):
    x = torch.randn(3, 9000, 70, device=gpu)
    codes = torch.randint(0, 70, (3, 9000), device=gpu)
    first = None
    for _ in range(3):
        xg = x.clone().requires_grad_(True)
        o, p = gs.code_balance(xg, codes), gs.code_log_probs(xg, codes, top=2)
        g, = torch.autograd.grad([o.loss, p.log_probs], xg, [torch.ones(3, device=gpu), torch.ones(3, 9000, device=gpu)])
        now = (o.loss, o.mean_probs, o.counts, p.log_probs, p.entropy, p.top_log_probs, g)
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


# ---- all three: differences, streams, the operators


@pytest.mark.parametrize("op", ["probs", "balance"])
def test_gradients_against_differences(gpu, op):
    """(L(x + hv) - L(x - hv)) / 2h: off by h^2 / 6 |L'''| and the roundings of L over h.  L is a sum of
    N rows of softmax terms with |v| <= 1 in every place: |L'''| <= 8 N (1 + log K) for weights in [0, 1];
    L's own terms are off by at most 1e-5 each."""
    N, K, h = 40, 30, 2.0 ** -5
    x = _logits((N,), K, F32, seed=1, spread=1.0).to(gpu)
    codes = torch.randint(0, K, (N,), generator=_gen(2)).to(gpu)
    v = (torch.rand(N, K, generator=_gen(3)) * 2 - 1).to(gpu)
    w = torch.rand(N, generator=_gen(4)).to(gpu)

    def L(x):
        if op == "probs":
            o = gs.code_log_probs(x, codes, top=2)
            return (o.log_probs.double() * w + o.entropy.double() * w + o.top_log_probs.double().sum(-1) * w).sum()
        o = gs.code_balance(x, codes)
        return o.loss.double() + (o.mean_probs.double() * w[:K]).sum()

    xg = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(L(xg), xg)
    slope = (g.double() * v).sum()
    diff = (L(x + h * v) - L(x - h * v)) / (2 * h)
    # (an alternative may change places within h: its log probability is continuous, the slope is not;
    # such rows are those whose second and third logit lie within 2h, and they are left out of the weights)
    if op == "probs":
        gap = x.topk(3, -1).values
        w[((gap[:, 1] - gap[:, 2]) <= 2 * h)] = 0.0
        xg = x.clone().requires_grad_(True)
        slope = (torch.autograd.grad(L(xg), xg)[0].double() * v).sum()
        diff = (L(x + h * v) - L(x - h * v)) / (2 * h)
    bound = h * h / 6 * 8 * 4 * N * (1 + math.log(K)) * 0.05 + 1e-5 * 4 * N / h * 0.05
    assert abs(float(slope - diff)) <= bound


def test_lookup_gradients_against_differences(gpu):
    """The output is linear in the codebook and in the scales: differences with h = 1 are exact up to roundings."""
    codes, book, s, grad = (t.to(gpu) for t in _lookup_inputs((500,), 40, 7, F32, seed=8))
    vb, vs = torch.randn(40, 7, generator=_gen(1)).to(gpu), torch.randn(500, generator=_gen(2)).to(gpu)

    def L(b, s):
        return (gs.lookup_codes(codes, b, s).double() * grad.double()).sum()

    b, sg = book.clone().requires_grad_(True), s.clone().requires_grad_(True)
    gb, g_s = torch.autograd.grad(L(b, sg), [b, sg])
    size = float((gs.lookup_codes(codes, book.abs() + vb.abs(), s + vs.abs()).double() * grad.double().abs()).sum())
    assert abs(float((gb.double() * vb).sum() - (L(book + vb, s) - L(book - vb, s)) / 2)) <= 64 * R.E * size
    assert abs(float((g_s.double() * vs).sum() - (L(book, s + vs) - L(book, s - vs)) / 2)) <= 64 * R.E * size


def test_other_stream(gpu):
    """Inputs made and outputs used on a stream that is not the default one."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        x = torch.randn(2000, 100, device=gpu).requires_grad_(True)
        book = torch.randn(100, 16, device=gpu).requires_grad_(True)
        o = gs.code_log_probs(x, top=1)
        codes = o.top_codes[:, 0]
        out = gs.lookup_codes(codes, book)
        bal = gs.code_balance(x, codes)
        (out.sum() + o.entropy.sum() + bal.loss).backward()
        got = [t.clone() for t in (codes, out.detach(), bal.counts, x.grad, book.grad)]
    side.synchronize()
    assert torch.equal(got[0].long(), x.detach().argmax(-1))
    assert torch.equal(got[1], book.detach()[got[0].long()])
    assert torch.equal(got[2], torch.bincount(got[0].long(), minlength=100).to(torch.int32))
    assert torch.equal(got[4], got[2].float()[:, None].expand(100, 16))
    assert bool(got[3].isfinite().all()) and bool(got[3].any())


def test_operators(gpu):
    """torch.ops.gsplat_hip.*: the same values as the Python calls, and their autograd formulas."""
    ops = torch.ops.gsplat_hip
    x = torch.randn(60, 30, device=gpu)
    codes = torch.randint(-1, 30, (60,), device=gpu)
    book = torch.randn(30, 5, device=gpu)
    s = torch.rand(60, device=gpu)

    def both(f, h, *leaves):
        res = []
        for fn in (f, h):
            ts = [t.clone().requires_grad_(True) for t in leaves]
            outs = fn(*ts)
            diff = [o for o in outs if o.is_floating_point() and o.requires_grad]
            grads = torch.autograd.grad([(o * o).sum() for o in diff], ts)
            res.append([*outs, *grads])
        for a, b in zip(*res):
            assert torch.equal(a, b)

    both(lambda b, s: [gs.lookup_codes(codes, b, s, 2.0)], lambda b, s: [ops.lookup_codes(codes, b, s, 2.0)], book, s)
    both(lambda x: list(gs.code_log_probs(x, codes, top=2)), lambda x: list(ops.code_log_probs(x, codes, 2, 1.0)[:4]), x)
    both(lambda x: list(gs.code_balance(x, codes)), lambda x: list(ops.code_balance(x, codes)[:3]), x)


def test_differentiated_once(gpu):
    """A gradient taken under create_graph says so when it is to be differentiated again."""
    x = torch.randn(20, 30, device=gpu, requires_grad=True)
    codes = torch.randint(0, 30, (20,), device=gpu)
    book = torch.randn(30, 4, device=gpu, requires_grad=True)
    for y, leaf in ((gs.lookup_codes(codes, book).square().sum(), book),
                    (gs.code_log_probs(x, codes, top=1).log_probs.square().sum(), x),
                    (gs.code_balance(x, codes).loss, x)):
        g, = torch.autograd.grad(y, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(g.sum(), leaf)


def test_inputs_that_are_not_plain(gpu):
    """Tensor subclasses take the operators and get the same values."""
    class Sub(torch.Tensor):
        pass

    x, codes = torch.randn(20, 30, device=gpu), torch.randint(0, 30, (20,), device=gpu)
    book = torch.randn(30, 4, device=gpu)
    assert torch.equal(gs.lookup_codes(codes, book.as_subclass(Sub)).as_subclass(torch.Tensor), gs.lookup_codes(codes, book))
    a, b = gs.code_log_probs(x.as_subclass(Sub), codes, top=2), gs.code_log_probs(x, codes, top=2)
    assert all(torch.equal(torch.Tensor(u) if u.is_floating_point() else u, v) for u, v in zip(a, b))
    a, b = gs.code_balance(x.as_subclass(Sub), codes), gs.code_balance(x, codes)
    assert torch.equal(a.counts, b.counts) and torch.equal(torch.Tensor(a.mean_probs), b.mean_probs)


def test_example_fits_a_scene(gpu):
    """examples/train_coded_scene.py: the three operators around the rasterizer, a scene that gets better."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_coded_scene.py")
    spec = importlib.util.spec_from_file_location("train_coded_scene", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    history, stored = example.train(steps=60, splats=1500, codes=32, size=128)
    assert bool(torch.isfinite(history["loss"]).all())
    assert float(history["mse"][-5:].mean()) < 0.3 * float(history["mse"][0])
    assert stored["codebook"].shape == (32, 3) and stored["codes"].shape == (1500,)
    assert int(history["used"][-1]) >= 4


def test_graph_capture(gpu):
    """All three, forward and backward, in a captured graph, replayed with new values between eager work."""
    x = torch.randn(3000, 200, device=gpu, requires_grad=True)
    book = torch.randn(200, 16, device=gpu, requires_grad=True)
    codes = torch.randint(-1, 200, (3000,), device=gpu)
    many = torch.randint(-1, 200, (20000,), device=gpu)

    def step():
        o, b = gs.code_log_probs(x, codes, top=3), gs.code_balance(x, codes)
        out, more = gs.lookup_codes(codes, book), gs.lookup_codes(many, book)
        outs = [o.log_probs, o.entropy, o.top_log_probs, b.loss, b.mean_probs, out, more]
        gx, gb = torch.autograd.grad(outs, [x, book], [torch.ones_like(t) for t in outs])
        return [*outs, o.top_codes, b.counts, gx, gb]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(3000, 200, generator=_gen(k)))
            codes.copy_(torch.randint(-1, 200, (3000,), generator=_gen(k + 9)))
            many.copy_(torch.randint(-1, 200, (20000,), generator=_gen(k + 19)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b.detach())


def test_lookup_of_more_vectors_than_a_launch_has_threads(gpu):
    """An output of 72 GiB: 2^32 vectors of 16 bytes and more."""
    N, D = 1 << 29, 72
    book = torch.randn(64, D, device=gpu).to(BF16)
    codes = torch.randint(0, 64, (N,), device=gpu, dtype=torch.int32)
    out = gs.lookup_codes(codes, book)
    for a in (0, N // 2 - 500, N // 9 * 8 - 500, N - 1000):
        assert torch.equal(out[a:a + 1000], book[codes[a:a + 1000].long()])
    del out
    torch.cuda.empty_cache()
