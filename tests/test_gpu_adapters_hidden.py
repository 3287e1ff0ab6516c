"""Hidden values of code_adapters keep their 32 bits on the way through the second product and the maps' gradients, in
16-bit types too: inputs whose large terms cancel, so that what is left shows the terms' own errors.  Against the 64-bit
formulas (oracle/decoders_reference.py), whose bounds leave a hidden value the roundings of its own sum and no others.

In 16 bits the factor that cancels is rounded, and what is left is 2^-9 (bfloat16) or 2^-12 (float16) of the terms at
most and next to nothing in some of the thousands of values: there a hidden value off by 2^-16 is past the bound."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R
from test_gpu_adapters import TYPES, _check
from test_gpu_decoders import BF16, F16, F32, _gen

pytestmark = pytest.mark.gpu

RANKS = [2, 8, 16, 18, 32, 48, 64, 66, 128]


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [200, 33000])
@pytest.mark.parametrize("r", [2, 8, 16, 17, 32, 64, 100])
def test_results_beside_a_base(gpu, dtype, r, N):
    """base is the map's result with the other sign, rounded; all ranks of a code are alike, and their errors add up."""
    K, D, E, g = 4, 3, 24, _gen(r)
    codes = torch.randint(0, K, (N,), generator=g).to(torch.int32)
    x = _normal(g, N, D, dtype=dtype)
    dn, up = (_normal(g, *s, dtype=dtype) for s in ((K, 1, D), (K, E, 1)))
    dn, up = dn.expand(K, r, D).contiguous(), up.expand(K, E, r).contiguous()
    alone = R.adapters(x, R.group(codes, K), dn, up, None, 0.75)["out"][0]
    _check(gpu, codes, x, dn, up, (-alone).to(dtype), torch.zeros(N, E, dtype=dtype), train=False)


def test_smaller_parts_of_both_factors(gpu):
    """float16: the hidden value's and the map's lower bits, multiplied."""
    r, t = 32, torch.float16
    x, dn, up = torch.tensor([[1 + 3 / 1024]], dtype=t), torch.full((1, r, 1), 1 + 4 / 1024, dtype=t), torch.full((1, 1, r), 1 + 7 / 1024, dtype=t)
    scale = 2.0 ** -5
    exact = scale * r * (1 + 3 / 1024) * (1 + 4 / 1024) * (1 + 7 / 1024)
    base = torch.tensor([[-exact]], dtype=t)
    _check(gpu, torch.zeros(1, dtype=torch.int32), x, dn, up, base, torch.zeros(1, 1, dtype=t), scale=scale, train=False)


def _gradients(gpu, codes, x, dn, up, go, scale):
    K = dn.shape[0]
    want = R.adapters(x, R.group(codes, K), dn, up, None, scale, False, go)
    leaves = [t.to(gpu).requires_grad_(True) for t in (x, dn, up)]
    out = gs.code_adapters(leaves[0], gs.group_codes(codes.to(gpu), K), *leaves[1:], scale=scale)
    return want, dict(zip(("g_rows", "g_down", "g_up"), torch.autograd.grad(out, leaves, go.to(gpu))))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r", RANKS)
def test_gradients_of_rows(gpu, dtype, r):
    """One row a code; half of its ranks against the other half."""
    K, D, E, g, scale = 100, 64, 3, _gen(r), 0.75
    half = r // 2
    codes = torch.randperm(K, generator=g).to(torch.int32)
    go = _normal(g, K, E, dtype=dtype)
    up = _normal(g, K, E, 2, dtype=dtype).repeat_interleave(half, 2)
    q = scale * (go.double()[:, None, :] @ up.double()[codes.long()])[:, 0]  # [K, r]: of each row
    ratio = torch.empty(K, 1, dtype=torch.float64)
    ratio[codes.long(), 0] = q[:, 0] / q[:, -1]
    one = _normal(g, K, D, dtype=dtype)
    other = (-ratio * one.double()).clamp(-1000, 1000).to(dtype)
    dn = torch.stack([one, other], 1).repeat_interleave(half, 1)
    want, got = _gradients(gpu, codes, _normal(g, K, D, dtype=dtype), dn, up, go, scale)
    R.check(got["g_rows"], want["g_rows"], f"r={r} {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r", RANKS)
def test_gradients_of_maps(gpu, dtype, r):
    """Two rows a code, one against the other: a row for down's gradient, a result's gradient for up's."""
    K, D, E, g, scale = 60, 64, 3, _gen(r), 0.75
    codes = torch.cat([torch.arange(K)] * 2).to(torch.int32)

    def against(first, a, b):
        """Rows with a * first + b * second near 0."""
        return torch.cat([first, (-(a / b)[:, None] * first.double()).clamp(-1000, 1000).to(dtype)])

    go, up = _normal(g, 2 * K, E, dtype=dtype), _normal(g, K, E, 1, dtype=dtype).expand(K, E, r).contiguous()
    q = (go.double()[:, None, :] @ up.double()[codes.long()])[:, 0, 0]
    x = against(_normal(g, K, D, dtype=dtype), q[:K], q[K:])
    want, got = _gradients(gpu, codes, x, _normal(g, K, r, D, dtype=dtype), up, go, scale)
    R.check(got["g_down"], want["g_down"], f"down r={r} {dtype}")
    x, dn = _normal(g, 2 * K, E, dtype=dtype), _normal(g, K, 1, E, dtype=dtype).expand(K, r, E).contiguous()
    h = (dn.double()[codes.long()] @ x.double()[..., None])[:, 0, 0]
    go = against(_normal(g, K, D, dtype=dtype), h[:K], h[K:])
    want, got = _gradients(gpu, codes, x, dn, _normal(g, K, D, r, dtype=dtype), go, scale)
    R.check(got["g_up"], want["g_up"], f"up r={r} {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,r", [(9, 70, 5), (61, 4096, 16), (700, 33, 24), (20000, 70, 100), (33000, 59, 8)])
def test_second_output_of_the_operator(gpu, dtype, N, D, r):
    """The hidden values, whatever their memory held before: those of rows without a code too."""
    K, E, g = 6, 40, _gen(N)
    codes = torch.randint(-1, K + 1, (N,), generator=g).to(torch.int32)  # (K: out of range)
    x, dn, up = _normal(g, N, D, dtype=dtype), _normal(g, K, r, D, dtype=dtype), _normal(g, K, E, r, dtype=dtype)
    order, _, starts = R.group(codes, K)
    named = int(starts[-1])
    n = order[:named].long()
    terms = dn.double()[codes[n].long()], x.double()[n, :, None]
    h = torch.zeros(N, r, dtype=torch.float64)
    size = h.clone()
    h[:named], size[:named] = (terms[0] @ terms[1])[..., 0], (terms[0].abs() @ terms[1].abs())[..., 0]
    groups = gs.group_codes(codes.to(gpu), K)
    maps = dn.to(gpu), up.to(gpu)
    for by_code in (False, True):
        rows = (x[order.long()] if by_code else x).to(gpu)
        for junk in (float("nan"), 7.0):
            held = [torch.full((N, r), junk, device=gpu) for _ in range(4)]
            del held
            hidden = torch.ops.gsplat_hip.code_adapters(rows, *groups, *maps, None, 1.0, by_code)[1]
            R.check(hidden, (h, 2 * (D + 4) * R.E * size), f"junk {junk}")
            assert not hidden[named:].any()
