"""Gradients of decoders by code against central differences of the forwards.

Every output is linear in each input by itself, so that a difference over any step is the slope but for roundings:
(L(x + hv) - L(x - hv)) / 2h is off by the forwards' own errors (the oracle's bounds, weighted) over h, and by the
rounding of x + hv, E of it, times the slope's weights.  v has the gradient's signs: the slope is the sum of the
gradient's sizes.  Every bound has to be below an eighth of it."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R
from test_gpu_decoders import _codes, _gen

pytestmark = pytest.mark.gpu

H = 0.5


def _compare(value, bounds, t, g, gpu, what):
    """value(t): in 64 bits; bounds(t): of its error; g: the gradient to check."""
    v = g.sign().float().cpu()
    up, down = t + H * v, t - H * v
    slope = float((g.double().cpu() * v).sum())
    diff = (value(up.to(gpu)) - value(down.to(gpu))) / (2 * H)
    moved = float((g.double().cpu().abs() * R.E * torch.maximum(up.abs(), down.abs()).double()).sum()) / H
    bound = 1.1 * (bounds(up) + bounds(down)) / (2 * H) + 2 * moved + 1e-6 * abs(slope)
    assert abs(slope - diff) <= bound, f"{what}: slope {slope}, difference {diff}, bound {bound}"
    assert bound <= abs(slope) / 8, f"{what}: slope {slope}, bound {bound}: a wrong gradient would pass"


@pytest.mark.parametrize("which", ["rows", "down", "up", "base"])
@pytest.mark.parametrize("N,K,D,E,r", [(60, 5, 20, 13, 4), (200, 9, 64, 48, 16), (3000, 7, 40, 72, 33)])
def test_adapters(gpu, which, N, K, D, E, r):
    g = _gen(N)
    codes = _codes((N,), K, seed=N)
    ts = {"rows": torch.randn(N, D, generator=g), "down": torch.randn(K, r, D, generator=g), "up": torch.randn(K, E, r, generator=g),
          "base": torch.randn(N, E, generator=g)}
    weight = torch.rand(N, E, generator=g) + 0.5
    groups, want_groups = gs.group_codes(codes.to(gpu), K), R.group(codes, K)

    def call(t):
        a = {k: (t if k == which else v.to(gpu)) for k, v in ts.items()}
        return gs.code_adapters(a["rows"], groups, a["down"], a["up"], a["base"], 0.6)

    def bounds(t):
        a = {**ts, which: t}
        return float((R.adapters(a["rows"], want_groups, a["down"], a["up"], a["base"], 0.6)["out"][1] * weight).sum())

    leaf = ts[which].to(gpu).requires_grad_(True)
    got, = torch.autograd.grad(call(leaf), leaf, weight.to(gpu))
    _compare(lambda t: float((call(t).double().cpu() * weight).sum()), bounds, ts[which], got, gpu, which)


@pytest.mark.parametrize("which", ["there", "rows", "weights"])
@pytest.mark.parametrize("N,S,K,D", [(50, 1, 4, 3), (300, 3, 11, 20), (5000, 2, 90, 48)])
def test_rows(gpu, which, N, S, K, D):
    g = _gen(N)
    codes = _codes((N, S), K, seed=N)
    groups, want_groups = gs.group_codes(codes.to(gpu), K, several=True), R.group(codes, K, True)
    x, rows, w = torch.randn(N, D, generator=g), torch.randn(N * S, D, generator=g), torch.rand(N, S, generator=g)
    t = {"there": x, "rows": rows, "weights": w}[which]
    weight = torch.rand((N * S if which == "there" else N), D, generator=g) + 0.5

    def call(t):
        if which == "there":
            return gs.rows_by_code(t, groups)
        return gs.rows_from_codes(t, groups, w.to(gpu)) if which == "rows" else gs.rows_from_codes(rows.to(gpu), groups, t)

    def bounds(t):
        want = R.by_code(t, want_groups) if which == "there" else \
            R.from_codes(t, want_groups, w) if which == "rows" else R.from_codes(rows, want_groups, t)
        return float((want["out"][1] * weight).sum())

    leaf = t.to(gpu).requires_grad_(True)
    got, = torch.autograd.grad(call(leaf), leaf, weight.to(gpu))
    _compare(lambda t: float((call(t).double().cpu() * weight).sum()), bounds, t, got, gpu, which)
