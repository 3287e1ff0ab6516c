"""The norm of many gradients together, and their clipping: what a training step over the tensors of a scene
(and of its codebooks and decoders) does between its backward pass and its optimizer.

torch.ops.gsplat_hip.{clip_gradients_, clip_gradients_into} are the same calls as operators.  The reference
has no counterpart.
"""
from __future__ import annotations

import math
from typing import Iterable, List, NamedTuple, Optional, Sequence, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, ptr, stream_of
from ._ops import _timed
from .codes import _NS, _check_device, _check_dtype, _check_size, _workspace


def _dense(t: Tensor) -> bool:
    """Whether t's values fill a piece of memory, in any order of its axes."""
    return torch.ops.aten.is_non_overlapping_and_dense(t)


class _Memory(NamedTuple):
    """Where a tensor's values lie, in bytes: pieces of `piece` adjacent ones, from `first` on, `axes` of them."""

    first: int
    piece: int
    axes: Tuple[Tuple[int, int], ...]  # (how many, how far apart), the farthest apart first

    @property
    def end(self) -> int:
        return self.first + self.piece + sum((n - 1) * s for n, s in self.axes)


def _memory(t: Tensor) -> _Memory:
    size = t.element_size()
    if t.is_contiguous():
        return _Memory(t.data_ptr(), t.numel() * size, ())
    # (values that are repeated lie in one place)
    axes = sorted(((n, s * size) for n, s in zip(t.shape, t.stride()) if n > 1 and s != 0), key=lambda a: -a[1])
    piece = size
    while axes and axes[-1][1] == piece:
        piece *= axes.pop()[0]
    return _Memory(t.data_ptr(), piece, tuple(axes))


_MOST_STEPS = 1 << 14


def _reaches(base: int, terms, lo: int, hi: int) -> bool:
    """Whether base + a sum of x * s over terms (s, least x, largest x) lies in [lo, hi] for some whole numbers x.

    The largest s first, since what the others can make up for leaves few x then; where the search is long all the same,
    True."""
    terms = sorted(terms, reverse=True)
    rest = [(0, 0, 0)]  # of the terms from k on: the least sum, the largest, what all sums are multiples of
    for s, a, b in reversed(terms):
        least, most, unit = rest[-1]
        rest.append((least + s * a, most + s * b, math.gcd(s, unit)))
    rest.reverse()
    steps = 0

    def search(k: int, at: int) -> bool:
        nonlocal steps
        steps += 1
        least, most, unit = rest[k]
        if steps > _MOST_STEPS:
            return True
        if at + most < lo or at + least > hi or (unit > 0 and lo + (at - lo) % unit > hi):
            return False
        if k == len(terms):
            return True
        s, a, b = terms[k]
        least, most, _ = rest[k + 1]
        a, b = max(a, -((at + most - lo) // s)), min(b, (hi - at - least) // s)
        return any(search(k + 1, at + x * s) for x in range(a, b + 1))

    return search(0, base)


def _meet(a: _Memory, b: _Memory) -> bool:
    """Whether two tensors have a byte in common."""
    if not a.axes and not b.axes:
        return a.first < b.end and b.first < a.end
    span = {}
    for n, s in a.axes:
        span[s] = (span.get(s, (0, 0))[0] - (n - 1), 0)
    for n, s in b.axes:
        least, most = span.get(s, (0, 0))
        span[s] = (least, most + n - 1)
    return _reaches(b.first - a.first, [(s, *x) for s, x in span.items()], 1 - b.piece, a.piece - 1)


def _repeats(t: Tensor) -> bool:
    """Whether two of a tensor's values have a byte in common."""
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        return True
    m = _memory(t)
    inner = m.piece
    for n, s in reversed(m.axes):
        if s < inner:  # (otherwise each step of an axis leaves all the inner ones behind)
            break
        inner += (n - 1) * s
    else:
        return False
    for k, (n, s) in enumerate(m.axes):  # the farthest axis where the two differ
        terms = [(s, 1, n - 1)] + [(t, 1 - i, i - 1) for i, t in m.axes[k + 1:]]
        if _reaches(0, terms, 1 - m.piece, m.piece - 1):
            return True
    return False


def _in_order(ranges) -> bool:
    """Whether of (first, end, written), sorted, none that is written overlaps another."""
    written = read = -1
    for first, end, mine in ranges:
        if first < max(written, read if mine else -1):
            return False
        if mine:
            written = max(written, end)
        else:
            read = max(read, end)
    return True


def _check_shared(gradients: Sequence[Tensor], out: Sequence[Tensor]) -> None:
    """What is written must be nobody else's, read or written (a tensor may be its own result)."""
    places, apart = [], []  # (memory, which, written); those that are their own results in another layout
    for k, (g, o) in enumerate(zip(gradients, out)):
        if o.numel() == 0:
            continue
        if not o.is_contiguous() and _repeats(o):
            raise ValueError("gradients that are written must not share memory with themselves")
        to, source = _memory(o), _memory(g)
        places.append((to, k, True))
        if source != to:
            places.append((source, k, False))
            if source.first == to.first:
                apart.append(k)
    places.sort(key=lambda p: (p[0].first, p[0].end))
    if not apart and _in_order((m.first, m.end, mine) for m, _, mine in places):
        return
    # Those whose extents overlap, together.
    group, end = [], 0
    for p in [*places, None]:
        if group and (p is None or p[0].first >= end):
            if not _separate(group, apart):
                raise ValueError("gradients that are written must not share memory")
            group, end = [], 0
        if p is not None:
            group.append(p)
            end = max(end, p[0].end)


def _separate(group, apart) -> bool:
    first = group[0][0]
    if all(m.axes == first.axes for m, _, _ in group) and not any(k in apart for _, k, _ in group):
        # Columns of one tensor: steps of the axes are longer than all of them together, so that pieces at the same
        # steps are what could overlap.
        inner = max(m.first + m.piece for m, _, _ in group) - first.first
        for n, s in reversed(first.axes):
            if s < inner:
                break
            inner += (n - 1) * s
        else:
            return _in_order((m.first, m.first + m.piece, mine) for m, _, mine in group)
    for i, (a, k, a_mine) in enumerate(group):
        for b, j, b_mine in group[i + 1:]:
            if b.first >= a.end:
                break
            if (a_mine or b_mine) and not (k == j and a.first == b.first) and _meet(a, b):
                return False
    return True


def _clip(gradients: Sequence[Tensor], out: Sequence[Tensor], max_norm: float) -> Tensor:
    """The C ABI's call; tensors that are not dense, or pairs of unequal layout, go through copies."""
    _check_clip(gradients, out, max_norm)
    like = gradients[0]
    table = (_lib.ClipTensor * len(gradients))()
    back, keep = [], []
    for entry, g, o in zip(table, gradients, out):
        source, to = g, o
        if not _dense(o) or o.stride() != g.stride():
            source, to = g.contiguous(), torch.empty_like(o, memory_format=torch.contiguous_format)
            back.append((o, to))
        keep.append((source, to))
        entry.source, entry.to, entry.size, entry.dtype = ptr(source), ptr(to), g.numel(), _lib.DTYPES[g.dtype]
    L = _lib.lib()
    norm = torch.empty((), dtype=torch.float32, device=like.device)
    n = L.gsplat_hip_clip_gradients_workspace_bytes(table, len(table))
    ws = _workspace(n, like)
    with torch.cuda.device(like.device), _timed("clip_gradients"):
        check(L.gsplat_hip_clip_gradients(table, len(table), max_norm, ptr(norm), ptr(ws), n, stream_of(like)),
              "gsplat_hip_clip_gradients")
    for o, to in back:
        o.copy_(to)
    return norm


@torch.library.custom_op(f"{_NS}::clip_gradients_", mutates_args=("gradients",))
def _clip_in_place(gradients: List[Tensor], max_norm: float) -> Tensor:
    return _clip(gradients, gradients, max_norm)


@torch.library.custom_op(f"{_NS}::clip_gradients_into", mutates_args=("out",))
def _clip_into(gradients: List[Tensor], out: List[Tensor], max_norm: float) -> Tensor:
    return _clip(gradients, out, max_norm)


@_clip_in_place.register_fake
def _(gradients, max_norm):
    return gradients[0].new_empty((), dtype=torch.float32)


@_clip_into.register_fake
def _(gradients, out, max_norm):
    return gradients[0].new_empty((), dtype=torch.float32)


def _check_reverse(tensors: Sequence[Tensor]) -> None:
    """There is no forward derivative; torch would leave a dual tensor's tangent as it is."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("clipping has no derivative: its tensors must have no tangent (not in forward mode)")


def _check_clip(gradients: Sequence[Tensor], out: Sequence[Tensor], max_norm: float) -> None:
    if not gradients:
        raise ValueError("at least one gradient is required")
    _check_size("gradients", len(gradients), _lib.MAX_TENSORS)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must be at least 0")
    if len(out) != len(gradients):
        raise ValueError("out must have a tensor for each gradient")
    for g, o in zip(gradients, out):
        _check_dtype("gradients", g)
        if g.requires_grad or o.requires_grad:
            raise ValueError("gradients and out must not require gradients themselves (detach them)")
        if o.dtype != g.dtype or o.shape != g.shape or o.device != g.device:
            raise ValueError("out must have the gradients' types, shapes and devices")
    _check_size("values in all", sum(g.numel() for g in gradients), _lib.MAX_VALUES)
    _check_device(**{f"gradients[{k}]": g for k, g in enumerate(gradients) if g.device != gradients[0].device},
                  gradients=gradients[0])
    _check_shared(gradients, out)


def clip_gradients(gradients: Iterable[Tensor], max_norm: float, out: Optional[Iterable[Tensor]] = None) -> Tensor:
    """Scales gradients by min(1, max_norm / norm), norm that of all of them together, and returns it.

    gradients: tensors of float32, bfloat16 or float16 and of any shapes on one device (None among them is
    left out).  out: where the results go; None: in place.  What is written shares no memory with another
    tensor, nor with itself (as what expand makes does).  The norm is a float32 tensor without axes; its
    squares are added in 64 bits.  max_norm=inf: the norm alone.  Where the norm is not finite (or
    past float32's range) the gradients stay as they are, and the norm says so.  A captured call keeps its max_norm."""
    gradients = gradients if isinstance(gradients, (list, tuple)) else list(gradients)
    out = out if out is None or isinstance(out, (list, tuple)) else list(out)
    if out is not None and len(out) != len(gradients):
        raise ValueError("out must have a tensor for each gradient")
    norm = _lib.host().clip_gradients(gradients, max_norm, out)
    if norm is not None:
        return norm
    out = None if out is None else [o for g, o in zip(gradients, out) if g is not None]
    gradients = [g for g in gradients if g is not None]
    _check_reverse(gradients if out is None else [*gradients, *out])
    _check_clip(gradients, gradients if out is None else out, max_norm)
    return _clip_in_place(gradients, float(max_norm)) if out is None else _clip_into(gradients, out, float(max_norm))
