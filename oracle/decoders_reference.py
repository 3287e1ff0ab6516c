"""Decoders by code and clipped gradients in plain 64-bit torch operations on the CPU, with bounds of what a
float32 computation rounded once to its output type may be off.

E is half a unit in the last place of float32.  A sum of n terms, in any order, each addition off by at
most 2 E (a matrix instruction's accumulation need not round to nearest): 2 (n + 4) E sum |terms|.

  adapters   hidden values h are such sums of D terms, and enter the second sum with all their bits.  Their
             errors add up through it at the weights of its terms.  (Where a factor is the sum of several
             16-bit floats, a matrix instruction adds many products before it rounds: a term's parts count
             as one addition.)
  clipping   the norm's squares are exact in 64 bits; it is rounded once, the factor once, the product once.

Every output is then rounded to its type: U[dtype] of its size, or half a denormal step.
"""
from __future__ import annotations

import math

import torch

from .codes_reference import E, U, _rounded, check  # noqa: F401

NAN = math.nan


def group(codes, K, several=False):
    """(order, places, starts) as int32."""
    flat = codes.reshape(-1).long()
    good = (flat >= 0) & (flat < K)
    keys = torch.where(good, flat, torch.full_like(flat, K))
    order = torch.sort(keys, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel())
    places = torch.where(good, places, torch.where(flat == -1, -1, -2))
    starts = torch.searchsorted(keys[order], torch.arange(K + 1))
    shape = codes.shape if several else (*codes.shape, 1)
    return order.to(torch.int32), places.reshape(shape).to(torch.int32), starts.to(torch.int32)


def _states(order, places):
    """Of each place: 1 a row, 0 none, NaN a code out of range."""
    at = places.reshape(-1)[order.long()]
    return torch.where(at >= 0, 1.0, torch.where(at == -1, 0.0, NAN)).double()


def by_code(rows, groups, grad=None):
    """{name: (value, bound)} of out and, with grad, of g_rows."""
    order, places, _ = groups
    S, D, dtype = places.shape[-1], rows.shape[-1], rows.dtype
    x = rows.reshape(-1, D).double()
    state = _states(order, places)
    out = torch.where(state[:, None] == 1, x[order.long() // S], 0 * state[:, None])
    r = {"out": (out, torch.zeros_like(out))}
    if grad is not None:
        r["g_rows"] = from_codes(grad, groups, None)["out"]
        r["g_rows"] = tuple(t.reshape(rows.shape) for t in r["g_rows"])
    return r


def from_codes(rows, groups, weights=None, grad=None):
    """{name: (value, bound)} of out and, with grad, of g_rows and g_weights."""
    order, places, _ = groups
    S, D, dtype = places.shape[-1], rows.shape[-1], rows.dtype
    at = places.reshape(-1, S).long()
    state = torch.where(at >= 0, 1.0, torch.where(at == -1, 0.0, NAN)).double()
    y = rows.double()[at.clamp(min=0)]
    y = torch.where(state[..., None] == 1, y, 0 * state[..., None])
    w = torch.ones(at.shape, dtype=torch.float64) if weights is None else weights.reshape(-1, S).double()
    terms = torch.where(state[..., None] == 0, 0.0, y * w[..., None])
    out = terms.sum(1)
    shape = (*places.shape[:-1], D)
    r = {"out": (out.reshape(shape), _rounded((S + 2) * E * terms.abs().sum(1).nan_to_num(0.0), out, dtype).reshape(shape))}
    if grad is not None:
        g = grad.reshape(-1, 1, D).double()
        lone = torch.where(state[..., None] == 1, g * w[..., None], 0 * state[..., None]).reshape(-1, D)[order.long()]
        r["g_rows"] = (lone, _rounded(4 * E * lone.abs().nan_to_num(0.0), lone, dtype))
        if weights is not None:
            gw = torch.where(state == 1, (g * y).sum(-1), 0 * state)
            size = (g * y).abs().sum(-1).nan_to_num(0.0)
            r["g_weights"] = (gw.reshape(weights.shape),
                              _rounded((D + 4) * E * size, gw, torch.float32).reshape(weights.shape))
    return r


def _product(a, da, b, db, n):
    """a @ b of 64-bit values with errors da, db of the factors: (value, bound) of a 32-bit sum of n terms."""
    v = a @ b
    bound = da @ b.abs() + a.abs() @ db + da @ db + 2 * (n + 4) * E * (a.abs() @ b.abs())
    return v, bound


def adapters(rows, groups, down, up, base=None, scale=1.0, by_code=False, grad=None):
    """{name: (value, bound)} of out and, with grad, of g_rows, g_down, g_up."""
    order, places, starts = groups
    dtype = rows.dtype
    K, r, D = down.shape
    Eo = up.shape[1]
    x = rows.reshape(-1, D).double()
    P = x.shape[0]
    dn, u = down.double(), up.double()
    out, d_out = torch.zeros(P, Eo, dtype=torch.float64), torch.zeros(P, Eo, dtype=torch.float64)
    b = torch.zeros(P, Eo, dtype=torch.float64) if base is None else base.reshape(-1, Eo).double()
    state = _states(order, places)
    where = torch.arange(P) if by_code else order.long()  # rows of the places
    out[where] = torch.where(state[:, None] == 1, out[where], 0 * state[:, None])
    train = grad is not None
    if train:
        g = grad.reshape(-1, Eo).double()
        gx, d_gx = torch.zeros_like(x), torch.zeros_like(x)
        gx[where] = torch.where(state[:, None] == 1, gx[where], 0 * state[:, None])
        g_down, d_down = torch.zeros_like(dn), torch.zeros_like(dn)
        g_up, d_up = torch.zeros_like(u), torch.zeros_like(u)
    zero = torch.zeros
    for k in range(K):
        n = where[int(starts[k]):int(starts[k + 1])]
        if n.numel() == 0:
            continue
        xs, m = x[n], n.numel()
        h, dh = _product(xs, zero(m, D).double(), dn[k].t(), zero(D, r).double(), D)
        y, dy = _product(h, dh, u[k].t(), zero(r, Eo).double(), r)
        out[n], d_out[n] = scale * y, abs(scale) * (dy + 2 * E * y.abs())
        if train:
            gs = g[n]
            q, dq = _product(gs, zero(m, Eo).double(), u[k], zero(Eo, r).double(), Eo)
            q, dq = scale * q, abs(scale) * (dq + 2 * E * q.abs())
            gx[n], d_gx[n] = _product(q, dq, dn[k], zero(r, D).double(), r)
            g_down[k], d_down[k] = _product(q.t(), dq.t(), xs, zero(m, D).double(), m)
            a, da = _product(gs.t(), zero(Eo, m).double(), h, dh, m)
            g_up[k], d_up[k] = scale * a, abs(scale) * (da + 2 * E * a.abs())
    total = out + b
    bound = _rounded(d_out + 2 * E * (out.abs() + b.abs()).nan_to_num(0.0), total, dtype)
    shape = (*rows.shape[:-1], Eo)
    res = {"out": (total.reshape(shape), bound.reshape(shape))}
    if train:
        res["g_rows"] = (gx.reshape(rows.shape), _rounded(d_gx, gx, dtype).reshape(rows.shape))
        res["g_down"] = (g_down, _rounded(d_down, g_down, dtype))
        res["g_up"] = (g_up, _rounded(d_up, g_up, dtype))
    return res


def clip(gradients, max_norm):
    """((norm, bound), [(out, bound)])"""
    total = sum(float(g.double().square().sum()) for g in gradients)
    norm = math.sqrt(total) if not math.isnan(total) else NAN
    if norm >= torch.finfo(torch.float32).max * (1 + E):  # (past what its float32 holds)
        norm = math.inf
    factor = min(1.0, max_norm / norm) if math.isfinite(norm) and norm > 0 else 1.0
    out = []
    for g in gradients:
        v = g.double() * factor
        bound = torch.zeros_like(v) if factor == 1.0 else _rounded(4 * E * v.abs().nan_to_num(0.0, 0.0, 0.0), v, g.dtype)
        out.append((v, bound))
    n = torch.tensor(norm, dtype=torch.float64)
    return (n, _rounded(1e-12 * n.abs().nan_to_num(0.0, 0.0), n, torch.float32)), out
