"""Gradients of log probabilities, entropy, best codes and balance against central differences of the forwards, in
the direction of the gradient's signs, where the slope is the sum of the gradient's sizes.

With |v| <= 1, p a row's distribution and k(..) its joint cumulants (|v - mean| <= 2, var v <= 1, E|v - mean| <= 1):
  (log p)'''  = -k(v,v,v),                  |k(v,v,v)| <= 2^3 / (6 sqrt 3) < 0.77
  (E_p a)'''  = k(a,v,v,v),                 |k(a,v,v,v)| <= R_a (E|v - mean|^3 + 3 E|v - mean| var v) <= 5 R_a
  (entropy)'''= -2 k(v,v,v) - k(z,v,v,v)
with R the range of a or of the logits z.  So (L(x + hv) - L(x - hv)) / 2h is off by at most h^2 / 6 of these, and by
the forwards' own errors (the oracle's bounds) over h.  The moved logits x + hv are rounded: by E |x + hv| each, times
the slope's weight |g| <= the row's, over h.  Every bound has to be below an eighth of the slope (entropies of wide
flat rows; the others lie below a twentieth): a gradient that is off by a quarter fails everywhere."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import codes_reference as R
from test_gpu_codes import F32, _gen, _logits

pytestmark = pytest.mark.gpu

H = 2.0 ** -6
CUBE = 0.77


def _compare(L, x, g, third, errors, gpu):
    """L: values in 64 bits of logits; g: the gradient to check; third, errors: sums of the bounds above."""
    v = g.sign().float().cpu()
    up, down = x + H * v, x - H * v
    slope = float((g.double().cpu() * v).sum())
    diff = (L(up.to(gpu)) - L(down.to(gpu))) / (2 * H)
    moved = float((g.double().cpu().abs() * R.E * torch.maximum(up.abs(), down.abs()).double()).sum()) / H
    bound = H * H / 6 * third + errors / H + 2 * moved
    assert abs(slope - diff) <= bound, f"slope {slope}, difference {diff}, bound {bound}"
    assert bound <= abs(slope) / 8, f"slope {slope}, bound {bound}: a wrong gradient would pass"


@pytest.mark.parametrize("what", ["log_probs", "entropy", "top_log_probs"])
@pytest.mark.parametrize("K", [7, 30, 300, 1100])
@pytest.mark.parametrize("T", [1.0, 2.0])
def test_probs(gpu, what, K, T):
    N, top = 60, 2
    x = _logits((N,), K, F32, seed=K, spread=1.0)
    codes = torch.randint(0, K, (N,), generator=_gen(2))
    w = torch.rand(N, generator=_gen(4)) + 0.5
    if what == "top_log_probs":
        # (a best code that changes places within h has a slope that does not: no weight)
        order = x.topk(top + 1, -1).values
        w[((order[:, :-1] - order[:, 1:]) <= 2.5 * H).any(-1)] = 0.0

    def value(t):
        out = getattr(gs.code_log_probs(t, codes.to(gpu), top=top, temperature=T), what).double().cpu()
        return float(((out.sum(-1) if what == "top_log_probs" else out) * w).sum())

    xg = x.to(gpu).requires_grad_(True)
    out = getattr(gs.code_log_probs(xg, codes.to(gpu), top=top, temperature=T), what)
    weights = (w[:, None].expand(N, top) if what == "top_log_probs" else w).to(gpu)
    g, = torch.autograd.grad(out, xg, weights.contiguous())
    span = (x.amax(-1) - x.amin(-1) + 2 * H).double() / T
    third = {"log_probs": CUBE * torch.ones(N), "entropy": 2 * CUBE + 5 * span, "top_log_probs": top * CUBE * torch.ones(N)}[what]
    bound = R.probs(x, codes, top, T)[what][1]
    bound = bound.sum(-1) if what == "top_log_probs" else bound
    _compare(value, x, g, float((third * w).sum()) / T ** 3, float((1.1 * bound * w).sum()), gpu)


@pytest.mark.parametrize("what", ["loss", "mean_probs"])
@pytest.mark.parametrize("B,G,K", [(1, 60, 7), (2, 50, 30), (1, 40, 300), (3, 20, 1100)])
def test_balance(gpu, what, B, G, K):
    x = _logits((B, G), K, F32, seed=K, spread=1.0)
    codes = torch.randint(0, K // 2, (B, G), generator=_gen(2))  # (one half of the codes: an uneven balance)
    w = torch.rand((B,) if what == "loss" else (B, K), generator=_gen(4)) + 0.5

    def value(t):
        return float((getattr(gs.code_balance(t, codes.to(gpu)), what).double().cpu() * w).sum())

    xg = x.to(gpu).requires_grad_(True)
    o = gs.code_balance(xg, codes.to(gpu))
    g, = torch.autograd.grad(getattr(o, what), xg, w.to(gpu))
    # a row's part of the value is E_p a / G
    a = w.double() if what == "mean_probs" else K * o.counts.cpu().double() / G * w[:, None].double()
    third = float((5 * (a.amax(-1) - a.amin(-1))).sum())  # (G rows of each image, over G)
    bound = R.balance(x, codes)[what][1]
    _compare(value, x, g, third, float((1.1 * bound * w).sum()), gpu)
