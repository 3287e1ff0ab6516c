"""The operators of scenes in codes in plain 64-bit torch operations on the CPU, with bounds of what a
float32 computation rounded once to its output type may be off.

E is half a unit in the last place of float32.  The bounds follow the formulas:

  logits     z = (x - max) / T has three roundings: |dz| <= 4 E |z|.  exp adds 4 E |z| (the argument of
             a base-2 exponential, rounded twice) and a few E of its own, so a probability's relative
             error is at most 8 E |z| + that of the sum.  The sum over K terms is made of chains of at most
             K / 16 + 32 additions.  log S lies in [0, log K], |z| <= |log p| + log K.
  lookup     products of three factors, sums of n of them in any order: (n + 4) E sum |terms|.

Every output is then rounded to its type: U[dtype] of its size, or half a denormal step.
"""
from __future__ import annotations

import math

import torch

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def _held(value, dtype):
    """value with what is past dtype's range as the infinity that dtype holds there."""
    big = torch.finfo(dtype).max * (1 + U[dtype])
    return torch.where(value.abs() >= big, torch.sign(value) * math.inf, value)


def _rounded(bound, value, dtype):
    return bound + U[dtype] * value.abs().nan_to_num(0.0, 0.0, 0.0) + TINY[dtype]


def lookup(codes, codebook, scales=None, factor=1.0, grad=None):
    """{name: (value, bound)} of out and, with grad, of g_codebook and g_scales."""
    dtype = codebook.dtype
    C, c = codebook.double(), codes.reshape(-1).long()
    K, D = C.shape
    N = c.numel()
    s = torch.ones(N, dtype=torch.float64) if scales is None else scales.reshape(-1).double()
    good = (c >= 0) & (c < K)
    rows = torch.zeros(N, D, dtype=torch.float64)
    rows[good] = C[c[good]]
    out = rows * (s * factor)[:, None]
    out[(c < -1) | (c >= K)] = math.nan
    shape = tuple(codes.shape)
    r = {"out": (out.reshape(*shape, D), _rounded(4 * E * out.abs().nan_to_num(0.0), out, dtype).reshape(*shape, D))}
    if grad is not None:
        g = grad.reshape(N, D).double()
        terms = g * (s * factor)[:, None]
        total, size = torch.zeros(K, D, dtype=torch.float64), torch.zeros(K, D, dtype=torch.float64)
        count = torch.zeros(K, dtype=torch.float64)
        total.index_add_(0, c[good], terms[good])
        size.index_add_(0, c[good], terms[good].abs())
        count.index_add_(0, c[good], torch.ones(int(good.sum()), dtype=torch.float64))
        r["g_codebook"] = (total, _rounded((count[:, None] + 4) * E * size, total, dtype))
        gs = factor * (g * rows).sum(-1)
        gs[(c < -1) | (c >= K)] = math.nan
        bound = (D + 4) * E * abs(factor) * (g * rows).abs().sum(-1)
        r["g_scales"] = (gs.reshape(shape), _rounded(bound, gs, torch.float32).reshape(shape))
    return r


def _distribution(x, T):
    """log p, p, whether a row has any logit, and the bound of log p, for 64-bit logits [N,K]."""
    K = x.shape[-1]
    m = x.amax(-1, keepdim=True)
    empty = m == -math.inf
    z = (x - torch.where(empty, torch.zeros_like(m), m)) / T
    lse = torch.logsumexp(z, -1, keepdim=True)
    lp = torch.where(empty, torch.full_like(z, -math.inf), z - lse)
    p = lp.exp()
    size = torch.where(lp.isfinite(), lp.abs(), torch.zeros_like(lp))
    d = E * (8 * size + 16 * math.log(K + 1) + K / 16 + 64)
    return lp, p, ~empty, d


def order(x):
    """Columns of each row, best first: the larger logit, NaN above all, the lower column among equal ones."""
    key = torch.where(x.isnan(), torch.full_like(x, math.inf), x)
    nan_first = torch.sort(key, dim=-1, descending=True, stable=True).indices
    # (NaN before +inf, each in the order of the columns)
    isnan = x.isnan().gather(-1, nan_first)
    again = torch.sort(isnan.to(torch.int8), dim=-1, descending=True, stable=True).indices
    return nan_first.gather(-1, again)


def probs(logits, codes=None, top=0, temperature=1.0, g_log_probs=None, g_entropy=None, g_top=None):
    """{name: (value, bound)}: log_probs, entropy, top_log_probs, top_codes (bound None), g_logits."""
    dtype, shape, K = logits.dtype, logits.shape[:-1], logits.shape[-1]
    x = logits.reshape(-1, K).double()
    N = x.shape[0]
    lp, p, some, d = _distribution(x, temperature)
    ent = torch.where(p > 0, -p * lp, torch.zeros_like(p))
    ent = torch.where(p.isnan(), p, ent)
    H = ent.sum(-1, keepdim=True)
    dH = ((p.nan_to_num(0.0) * (1 + lp.abs().nan_to_num(0.0, 0.0, 0.0)) * 2 * d).sum(-1, keepdim=True)
          + E * (K / 16 + 64) * (1 + math.log(K + 1)))
    i = torch.arange(N)
    r = {}
    if codes is not None:
        c = codes.reshape(-1).long()
        at = c.clamp(0, K - 1)
        bad = (c < -1) | (c >= K)
        v = torch.where(c >= 0, lp[i, at], torch.zeros(N, dtype=torch.float64))
        v = _held(torch.where(bad, torch.full_like(v, math.nan), v), torch.float32)
        r["log_probs"] = (v.reshape(shape), _rounded(d[i, at], v, torch.float32).reshape(shape))
    r["entropy"] = (H[:, 0].reshape(shape), _rounded(dH[:, 0], H[:, 0], torch.float32).reshape(shape))
    best = order(x)[:, :top]
    if top:
        v = _held(lp.gather(-1, best), torch.float32)
        r["top_log_probs"] = (v.reshape(*shape, top), _rounded(d.gather(-1, best), v, torch.float32).reshape(*shape, top))
        r["top_codes"] = (best.to(torch.int32).reshape(*shape, top), None)
    if g_log_probs is not None or g_entropy is not None or g_top is not None:
        w = torch.zeros(N, K, dtype=torch.float64)
        if g_log_probs is not None:
            c = codes.reshape(-1).long()
            ok = (c >= 0) & (c < K)
            w[i[ok], c[ok]] += g_log_probs.reshape(-1).double()[ok]
        if g_top is not None:
            w.scatter_add_(1, best, g_top.reshape(-1, top).double())
        ge = torch.zeros(N, 1, dtype=torch.float64) if g_entropy is None else g_entropy.reshape(-1, 1).double()
        total = w.sum(-1, keepdim=True)
        sized = w.abs().sum(-1, keepdim=True)
        lpf = torch.where(lp.isfinite(), lp, torch.zeros_like(lp))
        g = w - p * total - ge * p * (lpf + H)
        g = torch.where(some, g, torch.zeros_like(g)) / temperature
        bound = (p * sized * (d + (K + 8) * E) + ge.abs() * p * ((lpf.abs() + H) * (d + 8 * E) + d + dH)
                 + 8 * E * w.abs()) / temperature
        r["g_logits"] = (g.reshape(logits.shape), _rounded(bound.nan_to_num(0.0), g, dtype).reshape(logits.shape))
    return r


def balance(logits, codes, g_loss=None, g_mean=None):
    """{name: (value, bound)}: loss, counts (bound None), mean_probs, g_logits."""
    dtype, K = logits.dtype, logits.shape[-1]
    batched = logits.ndim == 3
    x = logits.double() if batched else logits.double()[None]
    B, G = x.shape[:2]
    c = codes.reshape(B, G, -1).long()
    out = {k: [] for k in ("loss", "counts", "mean_probs", "g_logits")}
    bounds = {k: [] for k in out}
    for b in range(B):
        part = ((c[b] >= 0) & (c[b] < K)).any(-1)
        given = c[b][(c[b] >= 0) & (c[b] < K)]
        bad = bool(((c[b] < -1) | (c[b] >= K)).any())
        counts = torch.bincount(given, minlength=K).double()
        lp, p, some, d = _distribution(x[b], 1.0) if G else (torch.zeros(0, K, dtype=torch.float64),) * 4
        p = torch.where(part[:, None], p, torch.zeros_like(p))
        rows, chosen = max(1, int(part.sum())), max(1, given.numel())
        mean = p.sum(0) / rows
        dmean = ((p * (2 * d + 4 * E)).sum(0) + G * E * p.sum(0)) / rows + 4 * E * mean
        share = counts / chosen
        loss = K * (share * mean).sum()
        out["loss"].append(torch.full_like(loss, math.nan) if bad else loss)
        bounds["loss"].append(K * (share * dmean).sum() + (K + 8) * E * loss)
        out["counts"].append(counts.to(torch.int32))
        out["mean_probs"].append(mean)
        bounds["mean_probs"].append(_rounded(dmean.nan_to_num(0.0), mean, torch.float32))
        if g_loss is not None or g_mean is not None:
            gl = 0.0 if g_loss is None else float(g_loss.reshape(B)[b])
            a = K * share * gl + (0.0 if g_mean is None else g_mean.reshape(B, K)[b].double())
            size = K * share * abs(gl) + (0.0 if g_mean is None else g_mean.reshape(B, K)[b].double().abs())
            dot = (p * a).sum(-1, keepdim=True)
            g = p * (a - dot) / rows
            bound = p * ((size + (p * size).sum(-1, keepdim=True)) * (2 * d + 8 * E)
                         + (p * size * (2 * d + (K + 8) * E)).sum(-1, keepdim=True)) / rows
            out["g_logits"].append(g)
            bounds["g_logits"].append(_rounded(bound.nan_to_num(0.0), g, dtype))
    r = {}
    for k in out:
        if out[k]:
            v = torch.stack(out[k])
            e = None if k == "counts" else torch.stack(bounds[k])
            r[k] = (v if batched else v[0], e if e is None or batched else e[0])
    return r


def check(got, want, what=""):
    """Asserts that got (a tensor) is within the bound of want = (value, bound); whole numbers equal."""
    value, bound = want
    got = got.detach().cpu()
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(value.shape)}"
    if bound is None:
        assert torch.equal(got, value), f"{what}: {(got != value).sum()} of {got.numel()} differ"
        return
    got = got.double()
    assert torch.equal(got.isnan(), value.isnan()), f"{what}: NaN at other places"
    plain = value.isfinite()
    assert torch.equal(got[~plain & ~value.isnan()], value[~plain & ~value.isnan()]), f"{what}: infinities"
    off = (got - value)[plain].abs() - bound[plain]
    assert off.numel() == 0 or float(off.max()) <= 0.0, \
        f"{what}: off by {float((got - value)[plain].abs().max()):.3g}, {float(off.max()):.3g} above its bound"
