"""The norm of many gradients together, and their clipping: what a training step over the tensors of a scene
(and of its codebooks and decoders) does between its backward pass and its optimizer.

torch.ops.gsplat_hip.{clip_gradients_, clip_gradients_into} are the same calls as operators.  The reference
has no counterpart.
"""
from __future__ import annotations

import ctypes
from typing import Iterable, List, Optional, Sequence

import torch
from torch import Tensor

from . import _lib
from ._lib import check, ptr, stream_of
from ._ops import _timed
from .codes import _NS, _check_device, _check_dtype, _check_size, _workspace


def _dense(t: Tensor) -> bool:
    """Whether t's values fill a piece of memory, in any order of its axes."""
    return torch.ops.aten.is_non_overlapping_and_dense(t)


def _range(t: Tensor):
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


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
    # What is written must be nobody else's, read or written (a tensor may be its own result).
    written = sorted(_range(o) for o in out if o.numel() and _dense(o))
    if any(a[1] > b[0] for a, b in zip(written, written[1:])):
        raise ValueError("gradients that are written must not share memory")
    w = 0
    for lo, hi in sorted(_range(g) for g, o in zip(gradients, out) if g.numel() and g.data_ptr() != o.data_ptr()):
        while w < len(written) and written[w][1] <= lo:
            w += 1
        if w < len(written) and written[w][0] < hi:
            raise ValueError("gradients that are written must not share memory")


def clip_gradients(gradients: Iterable[Tensor], max_norm: float, out: Optional[Iterable[Tensor]] = None) -> Tensor:
    """Scales gradients by min(1, max_norm / norm), norm that of all of them together, and returns it.

    gradients: tensors of float32, bfloat16 or float16 and of any shapes on one device (None among them is
    left out).  out: where the results go; None: in place.  The norm is a float32 tensor without axes; its
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
    _check_clip(gradients, gradients if out is None else out, max_norm)
    return _clip_in_place(gradients, float(max_norm)) if out is None else _clip_into(gradients, out, float(max_norm))
