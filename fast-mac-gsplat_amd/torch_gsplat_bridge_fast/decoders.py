"""Decoders by code: what belongs to a code, applied to the rows of the splats that name it.

  group_codes      splats' choices sorted by code
  rows_by_code     splats' rows in that order
  rows_from_codes  rows in that order back to their splats, weighted and summed
  code_adapters    a low-rank map of each splat's row by its code, beside a map that all share

A scene in codes (lookup_codes, code_log_probs, code_balance) gives every code a constant row.  Here a code
has a map of the splats' own features instead: groups = group_codes(codes, K), then

  one code per splat    code_adapters(features, groups, down, up, base=features @ shared)
  several, weighted     rows = rows_by_code(features, groups)
                        rows = code_adapters(rows, groups, down, up, by_code=True)   (or any map of one's own)
                        rows_from_codes(rows, groups, weights)

Codes are int32 or int64 of any shape.  -1 stands for no code: zeros, no gradient.  Any other value outside
[0, K) is a mistake that no call looks for, since that would wait for the device: nothing is read or written
for it, and what depends on it is NaN.

Rows and maps are float32, bfloat16 or float16; sums, hidden values and weights are float32, and results
and gradients are rounded once, to the type of what they belong to.  The last axis of rows is read in place
when its values are adjacent, whatever the rows' stride.  The same inputs give the same bits on every call.

torch.ops.gsplat_hip.{group_codes, rows_by_code, rows_from_codes, code_adapters} and their *_backward are
the same calls as operators, with fake implementations and autograd formulas.  The reference has no
counterpart.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, ptr, stream_of
from ._ops import _timed
from .codes import _NS, _check_codes, _check_device, _check_dtype, _check_given, _check_size, _rows_of, _stride, _workspace


class CodeGroups(NamedTuple):
    """What group_codes returns, all int32, for N splats of S choices each.

    Places past starts[K] hold the choices without a code, in their order.  (Groups of another making must be
    such a sort: values out of range are met by no access, but results that order leaves out are not written.)"""

    order: Tensor   # [N*S]: the choice at each place (splat * S + its number), by code and then in their order
    places: Tensor  # [..., S]: the place of each choice; -1 without a code, -2 with one out of range
    starts: Tensor  # [K+1]: code k's choices stand at places starts[k] .. starts[k+1]


# ---- the calls of the C ABI


@torch.library.custom_op(f"{_NS}::group_codes", mutates_args=())
def _group(codes: Tensor, num_codes: int, several: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """(order, places, starts)"""
    _check_group(codes, num_codes, several)
    c = codes.contiguous()
    i32 = dict(dtype=torch.int32, device=codes.device)
    order, starts = torch.empty((c.numel(),), **i32), torch.empty((num_codes + 1,), **i32)
    places = torch.empty(c.shape if several else (*c.shape, 1), **i32)
    meta = _lib.GroupMeta(c.numel(), num_codes, c.element_size())
    L = _lib.lib()
    n = L.gsplat_hip_group_codes_workspace_bytes(meta)
    ws = _workspace(n, c)
    with torch.cuda.device(c.device), _timed("group_codes"):
        check(L.gsplat_hip_group_codes(meta, ptr(c), ptr(order), ptr(places), ptr(starts), ptr(ws), n, stream_of(c)),
              "gsplat_hip_group_codes")
    return order, places, starts


@_group.register_fake
def _(codes, num_codes, several):
    i32 = dict(dtype=torch.int32)
    return (codes.new_empty((codes.numel(),), **i32), codes.new_empty(codes.shape if several else (*codes.shape, 1), **i32),
            codes.new_empty((num_codes + 1,), **i32))


def _rows_meta(flat: Tensor, places: Tensor) -> _lib.RowsMeta:
    S = places.shape[-1]
    return _lib.RowsMeta(places.numel() // S, S, flat.shape[-1], _stride(flat), _lib.DTYPES[flat.dtype])


def _named(starts: Tensor) -> int:
    """Where the number of choices with a code stands."""
    return ptr(starts) + 4 * (starts.numel() - 1)


@torch.library.custom_op(f"{_NS}::rows_by_code", mutates_args=())
def _by_code(rows: Tensor, order: Tensor, places: Tensor, starts: Tensor) -> Tensor:
    _check_by_code(rows, order, places, starts)
    flat, o, p, s = _rows_of(rows), order.contiguous(), places.contiguous(), starts.contiguous()
    out = torch.empty((o.numel(), rows.shape[-1]), dtype=rows.dtype, device=rows.device)
    with torch.cuda.device(rows.device), _timed("rows_by_code"):
        check(_lib.lib().gsplat_hip_rows_by_code(_rows_meta(flat, p), ptr(flat), ptr(o), ptr(p), _named(s), None,
                                                 ptr(out), stream_of(flat)), "gsplat_hip_rows_by_code")
    return out


@_by_code.register_fake
def _(rows, order, places, starts):
    return rows.new_empty((order.numel(), rows.shape[-1]))


def _by_code_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[1:])


def _by_code_grad(ctx, grad):
    return (_from_codes(grad, *ctx.saved_tensors, None) if ctx.needs_input_grad[0] else None), None, None, None


_by_code.register_autograd(_by_code_grad, setup_context=_by_code_setup)


@torch.library.custom_op(f"{_NS}::rows_from_codes", mutates_args=())
def _from_codes(rows: Tensor, order: Tensor, places: Tensor, starts: Tensor, weights: Optional[Tensor]) -> Tensor:
    _check_from_codes(rows, order, places, starts, weights)
    flat, p = _rows_of(rows), places.contiguous()
    w = None if weights is None else weights.contiguous()
    out = torch.empty((*places.shape[:-1], rows.shape[1]), dtype=rows.dtype, device=rows.device)
    with torch.cuda.device(rows.device), _timed("rows_from_codes"):
        check(_lib.lib().gsplat_hip_rows_from_codes(_rows_meta(flat, p), ptr(flat), ptr(p), ptr(w), ptr(out),
                                                    stream_of(flat)), "gsplat_hip_rows_from_codes")
    return out


@_from_codes.register_fake
def _(rows, order, places, starts, weights):
    return rows.new_empty((*places.shape[:-1], rows.shape[1]))


@torch.library.custom_op(f"{_NS}::rows_from_codes_backward", mutates_args=())
def _from_codes_backward(grad: Tensor, rows: Tensor, order: Tensor, places: Tensor, starts: Tensor,
                         weights: Optional[Tensor], need_rows: bool, need_weights: bool) -> Tuple[Tensor, Tensor]:
    _check_from_codes(rows, order, places, starts, weights)
    _check_given("grad", grad, (*places.shape[:-1], rows.shape[1]), rows.dtype, rows)
    if need_weights and weights is None:
        raise ValueError("weights are required for their gradient")
    flat, g, o, p, s = _rows_of(rows), *(t.contiguous() for t in (grad, order, places, starts))
    w = None if weights is None else weights.contiguous()
    g_rows = torch.empty(rows.shape if need_rows else (0,), dtype=rows.dtype, device=rows.device)
    g_weights = torch.empty(weights.shape if need_weights else (0,), dtype=torch.float32, device=rows.device)
    with torch.cuda.device(rows.device), _timed("rows_from_codes_backward"):
        check(_lib.lib().gsplat_hip_rows_from_codes_backward(
            _rows_meta(flat, p), ptr(g), ptr(flat), ptr(o), ptr(p), _named(s), ptr(w), ptr(g_rows) if need_rows else None,
            ptr(g_weights) if need_weights else None, stream_of(g)), "gsplat_hip_rows_from_codes_backward")
    return g_rows, g_weights


@_from_codes_backward.register_fake
def _(grad, rows, order, places, starts, weights, need_rows, need_weights):
    return (rows.new_empty(rows.shape if need_rows else (0,)),
            rows.new_empty(weights.shape if need_weights else (0,), dtype=torch.float32))


def _from_codes_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _from_codes_grad(ctx, grad):
    need = ctx.needs_input_grad
    g_rows, g_weights = _from_codes_backward(grad, *ctx.saved_tensors, need[0], need[4])
    return g_rows if need[0] else None, None, None, None, g_weights if need[4] else None


_from_codes.register_autograd(_from_codes_grad, setup_context=_from_codes_setup)


def _adapters_meta(flat: Tensor, down: Tensor, up: Tensor, scale: float, by_code: bool) -> _lib.AdaptersMeta:
    K, r, D = down.shape
    return _lib.AdaptersMeta(flat.shape[0], K, r, D, up.shape[1], _stride(flat), _lib.DTYPES[flat.dtype], int(by_code), scale)


@torch.library.custom_op(f"{_NS}::code_adapters", mutates_args=())
def _adapters(rows: Tensor, order: Tensor, places: Tensor, starts: Tensor, down: Tensor, up: Tensor,
              base: Optional[Tensor], scale: float, by_code: bool) -> Tuple[Tensor, Tensor]:
    """(out, hidden: float32 [rows, rank] in the order of the places, zeros at those without a code)"""
    _check_adapters(rows, order, places, starts, down, up, base, by_code)
    flat, o, p, s, dn, u = _rows_of(rows), *(t.contiguous() for t in (order, places, starts, down, up))
    b = None if base is None else base.contiguous()
    out = torch.empty((*rows.shape[:-1], up.shape[1]), dtype=rows.dtype, device=rows.device)
    hidden = torch.empty((flat.shape[0], down.shape[1]), dtype=torch.float32, device=rows.device)
    meta = _adapters_meta(flat, dn, u, scale, by_code)
    L = _lib.lib()
    n = L.gsplat_hip_code_adapters_workspace_bytes(meta)
    ws = _workspace(n, flat)
    with torch.cuda.device(rows.device), _timed("code_adapters"):
        check(L.gsplat_hip_code_adapters_forward(meta, ptr(flat), ptr(o), ptr(p), ptr(s), ptr(dn), ptr(u), ptr(b), ptr(out),
                                                 ptr(hidden), ptr(ws), n, stream_of(flat)),
              "gsplat_hip_code_adapters_forward")
    return out, hidden


@_adapters.register_fake
def _(rows, order, places, starts, down, up, base, scale, by_code):
    n = 1
    for s in rows.shape[:-1]:
        n = n * s
    return rows.new_empty((*rows.shape[:-1], up.shape[1])), rows.new_empty((n, down.shape[1]), dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::code_adapters_backward", mutates_args=())
def _adapters_backward(grad: Tensor, rows: Tensor, order: Tensor, places: Tensor, starts: Tensor, down: Tensor, up: Tensor,
                       hidden: Tensor, scale: float, by_code: bool, need_rows: bool, need_down: bool, need_up: bool
                       ) -> Tuple[Tensor, Tensor, Tensor]:
    _check_adapters(rows, order, places, starts, down, up, None, by_code)
    _check_given("grad", grad, (*rows.shape[:-1], up.shape[1]), rows.dtype, rows)
    _check_given("hidden", hidden, (order.numel(), down.shape[1]), torch.float32, rows)
    flat, g, o, p, s, dn, u, h = _rows_of(rows), *(t.contiguous() for t in (grad, order, places, starts, down, up, hidden))
    like = dict(dtype=rows.dtype, device=rows.device)
    g_rows, g_down, g_up = (torch.empty(t.shape if need else (0,), **like)
                            for t, need in ((rows, need_rows), (down, need_down), (up, need_up)))
    meta = _adapters_meta(flat, dn, u, scale, by_code)
    L = _lib.lib()
    n = L.gsplat_hip_code_adapters_backward_workspace_bytes(meta)
    ws = _workspace(n, flat)
    with torch.cuda.device(rows.device), _timed("code_adapters_backward"):
        check(L.gsplat_hip_code_adapters_backward(
            meta, ptr(g), ptr(flat), ptr(o), ptr(p), ptr(s), ptr(dn), ptr(u), ptr(h), ptr(g_rows) if need_rows else None,
            ptr(g_down) if need_down else None, ptr(g_up) if need_up else None, ptr(ws), n, stream_of(flat)),
            "gsplat_hip_code_adapters_backward")
    return g_rows, g_down, g_up


@_adapters_backward.register_fake
def _(grad, rows, order, places, starts, down, up, hidden, scale, by_code, need_rows, need_down, need_up):
    return (rows.new_empty(rows.shape if need_rows else (0,)), rows.new_empty(down.shape if need_down else (0,)),
            rows.new_empty(up.shape if need_up else (0,)))


def _adapters_setup(ctx, inputs, output):
    rows, order, places, starts, down, up, _, ctx.scale, ctx.by_code = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(rows, order, places, starts, down, up, output[1])


def _adapters_grad(ctx, grad, _):
    need = ctx.needs_input_grad
    g = (None, None, None)
    if need[0] or need[4] or need[5]:
        rows, order, places, starts, down, up, hidden = ctx.saved_tensors
        g = _adapters_backward(grad, rows, order, places, starts, down, up, hidden, ctx.scale, ctx.by_code, need[0], need[4],
                               need[5])
    return (g[0] if need[0] else None, None, None, None, g[1] if need[4] else None, g[2] if need[5] else None,
            grad if need[6] else None, None, None)


_adapters.register_autograd(_adapters_grad, setup_context=_adapters_setup)


# ---- checks


def _check_reverse(*tensors: Optional[Tensor]) -> None:
    """The operators have no forward derivative; torch would leave a dual input's tangent out."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("decoders by code have gradients in reverse mode only, not in forward mode")


def _check_group(codes: Tensor, num_codes: int, several: bool) -> None:
    _check_codes(codes)
    if num_codes < 1:
        raise ValueError("at least one code is required (num_codes >= 1)")
    _check_size("codes", num_codes, _lib.MAX_CODES)
    _check_size("choices", codes.numel(), _lib.MAX_ROWS)
    if several:
        if codes.ndim < 1 or codes.shape[-1] == 0:
            raise ValueError("codes must have a last axis of at least one choice per splat")
        _check_size("choices per splat", codes.shape[-1], _lib.MAX_CHOICES)
    _check_device(codes=codes)


def _check_groups(order: Tensor, places: Tensor, starts: Tensor) -> None:
    for name, t in (("order", order), ("places", places), ("starts", starts)):
        if t.dtype != torch.int32:
            raise ValueError(f"groups' {name} must be int32")
    if places.ndim < 1 or places.shape[-1] == 0 or tuple(order.shape) != (places.numel(),):
        raise ValueError("groups must be what group_codes returns: order [N*S], places [...,S]")
    if starts.ndim != 1 or starts.numel() < 2:
        raise ValueError("groups must be what group_codes returns: starts [K+1]")
    _check_size("choices", order.numel(), _lib.MAX_ROWS)
    _check_size("choices per splat", places.shape[-1], _lib.MAX_CHOICES)


def _check_rows(rows: Tensor) -> None:
    _check_dtype("rows", rows)
    if rows.ndim < 1 or rows.shape[-1] == 0:
        raise ValueError("rows must have a last axis of at least one value")
    _check_size("values per row", rows.shape[-1], _lib.MAX_CODE_WIDTH)


def _check_by_code(rows: Tensor, order: Tensor, places: Tensor, starts: Tensor) -> None:
    _check_rows(rows)
    _check_groups(order, places, starts)
    if rows.shape[:-1] != places.shape[:-1]:
        raise ValueError("rows must have a row per splat: the shape of the splats, and the values")
    _check_device(rows=rows, order=order, places=places, starts=starts)


def _check_from_codes(rows: Tensor, order: Tensor, places: Tensor, starts: Tensor, weights: Optional[Tensor]) -> None:
    _check_rows(rows)
    _check_groups(order, places, starts)
    if rows.ndim != 2 or rows.shape[0] != order.numel():
        raise ValueError("rows must have a row per choice, in the order of the codes")
    if weights is not None:
        if weights.dtype != torch.float32:
            raise ValueError("weights must be float32")
        if weights.shape != places.shape and (places.shape[-1] != 1 or weights.shape != places.shape[:-1]):
            raise ValueError("weights must match codes shape")
    _check_device(rows=rows, order=order, places=places, starts=starts, weights=weights)


def _check_adapters(rows: Tensor, order: Tensor, places: Tensor, starts: Tensor, down: Tensor, up: Tensor,
                    base: Optional[Tensor], by_code: bool) -> None:
    _check_rows(rows)
    _check_groups(order, places, starts)
    for name, t in (("down", down), ("up", up), ("base", base)):
        if t is not None and t.dtype != rows.dtype:
            raise ValueError(f"{name} must have the rows' type")
    if down.ndim != 3 or up.ndim != 3 or 0 in down.shape or 0 in up.shape:
        raise ValueError("down and up must have shapes [K,rank,D] and [K,E,rank], none of them 0")
    K, r, D = down.shape
    if up.shape[0] != K or up.shape[2] != r or rows.shape[-1] != D or starts.numel() != K + 1:
        raise ValueError("down [K,rank,D] and up [K,E,rank] must fit each other, the rows' D and the groups' K")
    _check_size("ranks", r, _lib.MAX_RANK)
    _check_size("values per result", up.shape[1], _lib.MAX_CODE_WIDTH)
    _check_size("codes", K, _lib.MAX_CODES)
    _check_size("values of all maps", K * r * max(D, up.shape[1]), _lib.MAX_VALUES)
    if by_code:
        if rows.ndim != 2 or rows.shape[0] != order.numel():
            raise ValueError("by_code: rows must have a row per choice, in the order of the codes")
    elif places.shape[-1] != 1:
        raise ValueError("several codes per splat: take the rows by code first (rows_by_code, by_code=True)")
    elif rows.shape[:-1] != places.shape[:-1]:
        raise ValueError("rows must have a row per splat: the shape of the codes, and the values")
    if base is not None and base.shape != (*rows.shape[:-1], up.shape[1]):
        raise ValueError("base must have the shape of the result")
    _check_device(rows=rows, order=order, places=places, starts=starts, down=down, up=up, base=base)


# ---- the public calls


def group_codes(codes: Tensor, num_codes: int, several: bool = False) -> CodeGroups:
    """The choices of all splats sorted by code.

    codes: one per splat, of any shape; several=True: the last axis holds a splat's choices.  The sort is
    stable, so that a code's choices keep their order; those without a code stand last.  The result is made
    once and serves rows_by_code, rows_from_codes and code_adapters, whatever their rows."""
    out = _lib.host().group_codes(codes, num_codes, several)
    if out is not None:
        return CodeGroups(*out)
    _check_group(codes, num_codes, several)
    return CodeGroups(*_group(codes, int(num_codes), bool(several)))


def rows_by_code(rows: Tensor, groups: CodeGroups) -> Tensor:
    """The splats' rows [..., D] in the order of their codes: [N*S, D], a copy for each choice.

    Code k's rows are starts[k] .. starts[k+1]; those past starts[K] are zeros (splats without a code).
    A row's gradient is the sum over the splat's choices, in their order."""
    out = _lib.host().rows_by_code(rows, *groups)
    if out is not None:
        return out
    _check_reverse(rows)
    _check_by_code(rows, *groups)
    return _by_code(rows, *groups)


def rows_from_codes(rows: Tensor, groups: CodeGroups, weights: Optional[Tensor] = None) -> Tensor:
    """Rows [N*S, D] in the order of the codes back to their splats: [..., D], the sum over a splat's choices.

    weights: float32 in the shape of the codes, or None for ones.  A choice without a code adds nothing (and
    gets no gradient).  Gradients flow to rows and weights."""
    out = _lib.host().rows_from_codes(rows, *groups, weights)
    if out is not None:
        return out
    _check_reverse(rows, weights)
    _check_from_codes(rows, *groups, weights)
    return _from_codes(rows, *groups, weights)


def code_adapters(rows: Tensor, groups: CodeGroups, down: Tensor, up: Tensor, base: Optional[Tensor] = None,
                  scale: float = 1.0, by_code: bool = False) -> Tensor:
    """base + scale * up[c] @ (down[c] @ row) for every splat's row, c its code: [..., E] from rows [..., D].

    down [K, rank, D] and up [K, E, rank]: a map of low rank for each code, the rank at most 128; base: what a
    map that all splats share made of the rows, or None for zeros.  One code per splat, or by_code=True: rows,
    base and the result stand in the order of the codes, [N*S, D], as rows_by_code leaves them.  A splat
    without a code gets base.  Gradients flow to rows, down, up and base; codes that no splat names get zeros."""
    out = _lib.host().code_adapters(rows, *groups, down, up, base, scale, by_code)
    if out is not None:
        return out
    _check_reverse(rows, down, up, base)
    _check_adapters(rows, *groups, down, up, base, by_code)
    return _adapters(rows, *groups, down, up, base, float(scale), bool(by_code))[0]
