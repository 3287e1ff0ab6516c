"""Log probabilities and balance of logits far from zero and at small temperatures: rows masked wholly with a
finite value, unnormalised distances, annealed temperatures.  The widths take every kind of kernel: rows of 2 to
64 lanes, of a workgroup, of several workgroups; in the balance rows of one and of several wavefronts and rows
that are read twice.  Values and bounds: oracle/codes_reference.py."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import codes_reference as R
from test_gpu_codes import BF16, F16, F32, _check_balance, _gen, _logits

pytestmark = pytest.mark.gpu

# largest logits from those whose exponents are held exactly to the types' limits
FAR = [1e5, 3e6, 1e7, 1e9, 1e10, 1e13, 1e15, 1e20, 1e29, 1e31, 3e38]


def _far_rows(K, dtype):
    """Rows of one far value, of far values a step apart, and of near logits with far ones among them."""
    limit = float(torch.finfo(dtype).max)
    rows = []
    g = _gen(K)
    for far in FAR:
        for v in (far, -far):
            if far > limit:
                continue
            rows.append(torch.full((K,), v))
            near = torch.full((K,), v)
            near[torch.rand(K, generator=g) < 0.5] = v * (1 - 2.0 ** -7)
            rows.append(near)
            if v < 0:
                masked = torch.randn(K, generator=g)
                masked[torch.rand(K, generator=g) < 0.5] = v
                rows.append(masked)
    return torch.stack(rows).to(dtype)


def _check(gpu, x, codes, top, T, what):
    """As test_gpu_codes._check_probs, with gradients of the outputs of the temperature's size."""
    g = _gen(5)
    n = x.shape[0]
    gl, ge, gt = (T * torch.randn(s, generator=g) for s in ((n,), (n,), (n, top)))
    want = R.probs(x, codes, top, T, gl, ge, gt)
    xg = x.to(gpu).requires_grad_(True)
    o = gs.code_log_probs(xg, codes.to(gpu), top=top, temperature=T)
    for k in ("log_probs", "entropy", "top_codes", "top_log_probs"):
        R.check(getattr(o, k), want[k], f"{what} {k}")
    got, = torch.autograd.grad([o.log_probs, o.entropy, o.top_log_probs], xg, [t.to(gpu) for t in (gl, ge, gt)])
    R.check(got, want["g_logits"], f"{what} g_logits")


PROBS_KS = [4, 6, 64, 70, 250, 300, 1000, 1500, 2500, 9000, 20000]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K", PROBS_KS)
@pytest.mark.parametrize("T", [1.0, 0.3])
def test_probs_far_from_zero(gpu, dtype, K, T):
    x = _far_rows(K, dtype)
    codes = torch.randint(-1, K, (x.shape[0],), generator=_gen(K))
    for top in (1, 3):
        _check(gpu, x, codes, top, T, f"K={K} {dtype} T={T} top={top}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("K", PROBS_KS)
@pytest.mark.parametrize("T", [1e-5, 1e-6, 1e-7, 1e-9, 1e-20])
def test_probs_of_small_temperatures(gpu, dtype, K, T):
    x = _logits((7,), K, dtype, seed=K, masked=0.1)
    x[1] = x[0, 0].abs() + 1.0                     # equal logits
    x[2, : K // 2] = x[2].abs().max() + 0.5        # several best ones
    x[3] = float(torch.finfo(dtype).min)
    codes = torch.randint(-1, K, (7,), generator=_gen(K))
    for top in (1, 3):
        _check(gpu, x, codes, top, T, f"K={K} {dtype} T={T} top={top}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K", [4, 6, 70, 300, 1500, 3000, 5000, 9000, 16000, 20000])
def test_balance_far_from_zero(gpu, dtype, K):
    x = _far_rows(K, dtype)
    codes = torch.randint(0, K, (x.shape[0],), generator=_gen(K))
    _check_balance(gpu, x, codes, what=f"K={K} {dtype}")
    # one such row among ordinary ones, and one image with and one without it
    y = torch.stack([_logits((40,), K, dtype, seed=K + b) for b in range(2)])
    y[1, 7] = -1e10
    _check_balance(gpu, y, torch.randint(-1, K, (2, 40), generator=_gen(K)), what=f"K={K} {dtype} one row")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K", PROBS_KS)
@pytest.mark.parametrize("T", [2.0, 1e6, 1e30])
def test_probs_of_rows_that_span_the_range(gpu, dtype, K, T):
    """Logits at both ends of the type: their difference is past the range, over T it is not."""
    big = float(torch.finfo(dtype).max)
    x = torch.randn(6, K, generator=_gen(K)).to(dtype)
    x[0, ::2], x[0, 1::2] = big, -big
    x[1, 0] = -big
    x[2] = -big
    x[2, K - 1] = big
    x[3] = torch.linspace(-0.9, 0.9, K).mul(big).to(dtype)
    x[4, : K // 2] = 0.75 * big
    x[5, K // 2] = big
    codes = torch.tensor([1, 0, 0, K // 2, K - 1, K // 2])
    _check(gpu, x, codes, 3, T, f"K={K} {dtype} T={T}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("K", PROBS_KS)
@pytest.mark.parametrize("T", [1e-30, 1e3, 1e10, 1e30])
def test_probs_of_extreme_temperatures(gpu, dtype, K, T):
    x = _logits((5,), K, dtype, seed=K, masked=0.1)
    x[1] = 1.5
    _check(gpu, x, torch.randint(-1, K, (5,), generator=_gen(K)), 3, T, f"K={K} {dtype} T={T}")
