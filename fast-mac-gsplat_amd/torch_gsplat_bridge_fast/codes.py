"""Scenes in codes: splats that name rows of a learned codebook instead of owning their attributes.

  lookup_codes     attributes of splats from their codes, and the codebook's gradient
  code_log_probs   log probabilities of codes (the rate of a scene), the entropy of each splat's
                   choice and its likeliest codes (the first is the assignment itself)
  code_balance     how evenly the codes are used: counts, mean probabilities and a loss

A training step with them: logits of every splat over the codes -> code_log_probs picks the codes ->
lookup_codes makes the attributes -> the rasterizer's image and its loss, plus the rate and the balance
(examples/train_coded_scene.py).

Codes are int32 or int64, [G] or [B,G] like the splats' other attributes (lookup_codes and
code_log_probs take any number of leading axes).  -1 stands for no code: the splat's attributes, log
probability and gradients are zero and it is not counted.  Any other value outside [0, K) is a mistake
that no call looks for, since that would wait for the device: nothing is read, written or counted for
it, and the outputs that depend on it are NaN.

Codebooks and logits are float32, bfloat16 or float16; sums, probabilities, scales and losses are
float32, and gradients are rounded once, to the type of what they belong to.  The last axis of a
codebook or of logits is read in place when its values are adjacent, whatever the rows' stride (a
column range of a wider codebook, say).  The same inputs give the same bits on every call: no sum's
order depends on the run.

torch.ops.gsplat_hip.{lookup_codes, code_log_probs, code_balance} and their *_backward are the same
calls as operators, with fake implementations and autograd formulas.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, ptr, stream_of
from ._ops import _timed

_NS = "gsplat_hip"


class CodeLogProbs(NamedTuple):
    """What code_log_probs returns; a field that was not asked for is None."""

    log_probs: Optional[Tensor]      # float32, the shape of the codes
    entropy: Tensor                  # float32, in nats
    top_log_probs: Optional[Tensor]  # float32 [..., top]
    top_codes: Optional[Tensor]      # int32 [..., top], best first


class CodeBalance(NamedTuple):
    """What code_balance returns: [B] and [B,K], or [] and [K] without a batch axis."""

    loss: Tensor        # float32
    counts: Tensor      # int32
    mean_probs: Tensor  # float32


# ---- the calls of the C ABI


def _rows_of(x: Tensor) -> Tensor:
    """x as [N, C] with adjacent values in a row, copied only where it has to be."""
    C = x.shape[-1]
    try:
        flat = x.view(-1, C) if x.numel() else x.reshape(-1, C) if C else x.new_empty((0, 0))
    except RuntimeError:
        flat = x.contiguous().view(-1, C)
    if flat.shape[0] > 1 and flat.stride(0) < C or C > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    return flat


def _stride(flat: Tensor) -> int:
    return flat.stride(0) if flat.shape[0] > 1 else flat.shape[1]


def _lookup_meta(codes: Tensor, codebook: Tensor, factor: float) -> _lib.LookupMeta:
    return _lib.LookupMeta(codes.numel(), codebook.shape[0], codebook.shape[1], _stride(codebook),
                           _lib.DTYPES[codebook.dtype], codes.element_size(), factor)


def _workspace(n: int, like: Tensor) -> Tensor:
    return torch.empty((max(n, 1),), dtype=torch.uint8, device=like.device)


@torch.library.custom_op(f"{_NS}::lookup_codes", mutates_args=())
def _lookup(codes: Tensor, codebook: Tensor, scales: Optional[Tensor], factor: float) -> Tensor:
    _check_lookup(codes, codebook, scales)
    book, c = _rows_of(codebook), codes.contiguous()
    s = None if scales is None else scales.contiguous()
    out = torch.empty((*codes.shape, codebook.shape[1]), dtype=codebook.dtype, device=codebook.device)
    with torch.cuda.device(codebook.device), _timed("lookup_codes"):
        check(_lib.lib().gsplat_hip_lookup_forward(_lookup_meta(c, book, factor), ptr(c), ptr(book), ptr(s), ptr(out),
                                                   stream_of(out)), "gsplat_hip_lookup_forward")
    return out


@_lookup.register_fake
def _(codes, codebook, scales, factor):
    return codebook.new_empty((*codes.shape, codebook.shape[1]))


@torch.library.custom_op(f"{_NS}::lookup_codes_backward", mutates_args=())
def _lookup_backward(grad: Tensor, codes: Tensor, codebook: Tensor, scales: Optional[Tensor], factor: float,
                     need_codebook: bool, need_scales: bool) -> Tuple[Tensor, Tensor]:
    _check_lookup(codes, codebook, scales)
    _check_given("grad", grad, (*codes.shape, codebook.shape[1]), codebook.dtype, codes)
    book, c, g = _rows_of(codebook), codes.contiguous(), grad.contiguous()
    s = None if scales is None else scales.contiguous()
    meta = _lookup_meta(c, book, factor)
    L = _lib.lib()
    g_book = torch.empty(codebook.shape if need_codebook else (0,), dtype=book.dtype, device=book.device)
    g_scales = torch.empty(codes.shape if need_scales else (0,), dtype=torch.float32, device=book.device)
    n = L.gsplat_hip_lookup_backward_workspace_bytes(meta) if need_codebook else 0
    ws = _workspace(n, book)
    with torch.cuda.device(book.device), _timed("lookup_codes_backward"):
        check(L.gsplat_hip_lookup_backward(meta, ptr(g), ptr(c), ptr(book), ptr(s), ptr(g_book) if need_codebook else None,
                                           ptr(g_scales) if need_scales else None, ptr(ws), n, stream_of(g)),
              "gsplat_hip_lookup_backward")
    return g_book, g_scales


@_lookup_backward.register_fake
def _(grad, codes, codebook, scales, factor, need_codebook, need_scales):
    return (codebook.new_empty(codebook.shape if need_codebook else (0,)),
            codebook.new_empty(codes.shape if need_scales else (0,), dtype=torch.float32))


def _lookup_setup(ctx, inputs, output):
    codes, codebook, scales, ctx.factor = inputs
    ctx.save_for_backward(codes, codebook, scales)


def _lookup_grad(ctx, grad):
    codes, codebook, scales = ctx.saved_tensors
    need = ctx.needs_input_grad
    g_book, g_scales = _lookup_backward(grad, codes, codebook, scales, ctx.factor, need[1], need[2])
    return None, g_book if need[1] else None, g_scales if need[2] else None, None


_lookup.register_autograd(_lookup_grad, setup_context=_lookup_setup)


def _probs_meta(flat: Tensor, codes: Optional[Tensor], top: int, temperature: float) -> _lib.ProbsMeta:
    return _lib.ProbsMeta(flat.shape[0], flat.shape[1], top, _stride(flat), _lib.DTYPES[flat.dtype],
                          4 if codes is None else codes.element_size(), temperature)


@torch.library.custom_op(f"{_NS}::code_log_probs", mutates_args=())
def _probs(logits: Tensor, codes: Optional[Tensor], top: int, temperature: float
           ) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(log_probs (empty without codes), entropy, top_log_probs, top_codes, row_stats)"""
    _check_probs(logits, codes, top, temperature)
    flat = _rows_of(logits)
    c = None if codes is None else codes.contiguous()
    shape = logits.shape[:-1]
    f32 = dict(dtype=torch.float32, device=logits.device)
    log_probs = torch.empty(shape if c is not None else (0,), **f32)
    entropy = torch.empty(shape, **f32)
    top_log_probs = torch.empty((*shape, top), **f32)
    top_codes = torch.empty((*shape, top), dtype=torch.int32, device=logits.device)
    stats = torch.empty((*shape, 2), **f32)
    meta = _probs_meta(flat, c, top, temperature)
    L = _lib.lib()
    n = L.gsplat_hip_code_probs_workspace_bytes(meta)
    ws = _workspace(n, flat)
    with torch.cuda.device(flat.device), _timed("code_log_probs"):
        check(L.gsplat_hip_code_probs_forward(meta, ptr(flat), ptr(c), ptr(log_probs) if c is not None else None,
                                              ptr(entropy), ptr(top_log_probs), ptr(top_codes), ptr(stats), ptr(ws), n,
                                              stream_of(flat)), "gsplat_hip_code_probs_forward")
    return log_probs, entropy, top_log_probs, top_codes, stats


@_probs.register_fake
def _(logits, codes, top, temperature):
    shape = logits.shape[:-1]
    f32 = dict(dtype=torch.float32)
    return (logits.new_empty(shape if codes is not None else (0,), **f32), logits.new_empty(shape, **f32),
            logits.new_empty((*shape, top), **f32), logits.new_empty((*shape, top), dtype=torch.int32),
            logits.new_empty((*shape, 2), **f32))


@torch.library.custom_op(f"{_NS}::code_log_probs_backward", mutates_args=())
def _probs_backward(g_log_probs: Optional[Tensor], g_entropy: Optional[Tensor], g_top: Optional[Tensor], logits: Tensor,
                    codes: Optional[Tensor], top_codes: Tensor, stats: Tensor, entropy: Tensor, temperature: float
                    ) -> Tensor:
    shape, f32 = tuple(logits.shape[:-1]), torch.float32
    _check_probs(logits, codes, top_codes.shape[-1] if top_codes.ndim else 0, temperature)
    many = (*shape, top_codes.shape[-1] if top_codes.ndim else 0)
    for name, t, given, dtype in (("g_log_probs", g_log_probs if codes is not None else None, shape, f32),
                                  ("g_entropy", g_entropy, shape, f32), ("g_top", g_top, many, f32),
                                  ("top_codes", top_codes, many, torch.int32), ("stats", stats, (*shape, 2), f32),
                                  ("entropy", entropy, shape, f32)):
        _check_given(name, t, given, dtype, logits)
    flat = _rows_of(logits)
    c = None if codes is None else codes.contiguous()
    top_codes, stats, entropy = top_codes.contiguous(), stats.contiguous(), entropy.contiguous()
    g = [None if t is None else t.contiguous() for t in (g_log_probs if c is not None else None, g_entropy, g_top)]
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    top = top_codes.shape[-1]
    if top == 0:
        g[2] = None
    with torch.cuda.device(flat.device), _timed("code_log_probs_backward"):
        check(_lib.lib().gsplat_hip_code_probs_backward(
            _probs_meta(flat, c, top, temperature), ptr(flat), ptr(c), ptr(top_codes), ptr(stats), ptr(entropy),
            ptr(g[0]), ptr(g[1]), ptr(g[2]), ptr(out), stream_of(flat)), "gsplat_hip_code_probs_backward")
    return out


@_probs_backward.register_fake
def _(g_log_probs, g_entropy, g_top, logits, codes, top_codes, stats, entropy, temperature):
    return logits.new_empty(logits.shape)


def _probs_setup(ctx, inputs, output):
    logits, codes, _, ctx.temperature = inputs
    _, entropy, _, top_codes, stats = output
    ctx.mark_non_differentiable(top_codes, stats)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(logits, codes, top_codes, stats, entropy)


def _probs_grad(ctx, g_log_probs, g_entropy, g_top, *_):
    logits, codes, top_codes, stats, entropy = ctx.saved_tensors
    g = None
    if ctx.needs_input_grad[0]:
        g = _probs_backward(g_log_probs, g_entropy, g_top, logits, codes, top_codes, stats, entropy, ctx.temperature)
    return g, None, None, None


_probs.register_autograd(_probs_grad, setup_context=_probs_setup)


def _balance_meta(flat: Tensor, B: int, choices: int, code_bytes: int) -> _lib.BalanceMeta:
    return _lib.BalanceMeta(flat.shape[0] // B, B, flat.shape[1], choices, _lib.DTYPES[flat.dtype], _stride(flat),
                            code_bytes)


@torch.library.custom_op(f"{_NS}::code_balance", mutates_args=())
def _balance(logits: Tensor, codes: Tensor) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(loss, counts, mean_probs, row_stats, totals)"""
    _check_balance(logits, codes)
    flat, c = _rows_of(logits), codes.contiguous()
    batch, K = logits.shape[:-2], logits.shape[-1]
    B = batch[0] if batch else 1
    f32 = dict(dtype=torch.float32, device=logits.device)
    i32 = dict(dtype=torch.int32, device=logits.device)
    loss, counts, mean = torch.empty(batch, **f32), torch.empty((*batch, K), **i32), torch.empty((*batch, K), **f32)
    stats, totals = torch.empty((*logits.shape[:-1], 2), **f32), torch.empty((B, 4), **i32)
    meta = _balance_meta(flat, B, codes.shape[-1] if codes.ndim == logits.ndim else 1, c.element_size())
    L = _lib.lib()
    n = L.gsplat_hip_code_balance_workspace_bytes(meta)
    ws = _workspace(n, flat)
    with torch.cuda.device(flat.device), _timed("code_balance"):
        check(L.gsplat_hip_code_balance_forward(meta, ptr(flat), ptr(c), ptr(loss), ptr(counts), ptr(mean), ptr(stats),
                                                ptr(totals), ptr(ws), n, stream_of(flat)),
              "gsplat_hip_code_balance_forward")
    return loss, counts, mean, stats, totals


@_balance.register_fake
def _(logits, codes):
    batch, K = logits.shape[:-2], logits.shape[-1]
    f32, i32 = dict(dtype=torch.float32), dict(dtype=torch.int32)
    return (logits.new_empty(batch, **f32), logits.new_empty((*batch, K), **i32), logits.new_empty((*batch, K), **f32),
            logits.new_empty((*logits.shape[:-1], 2), **f32), logits.new_empty((batch[0] if batch else 1, 4), **i32))


@torch.library.custom_op(f"{_NS}::code_balance_backward", mutates_args=())
def _balance_backward(g_loss: Optional[Tensor], g_mean: Optional[Tensor], logits: Tensor, counts: Tensor, stats: Tensor,
                      totals: Tensor) -> Tensor:
    _check_logits(logits)
    _check_images(logits)
    batch, K, f32 = tuple(logits.shape[:-2]), logits.shape[-1], torch.float32
    for name, t, given, dtype in (("g_loss", g_loss, batch, f32), ("g_mean", g_mean, (*batch, K), f32),
                                  ("counts", counts, (*batch, K), torch.int32),
                                  ("stats", stats, (*logits.shape[:-1], 2), f32),
                                  ("totals", totals, (batch[0] if batch else 1, 4), torch.int32)):
        _check_given(name, t, given, dtype, logits)
    _check_device(logits=logits)
    flat = _rows_of(logits)
    g = [None if t is None else t.contiguous() for t in (g_loss, g_mean)]
    counts, stats, totals = counts.contiguous(), stats.contiguous(), totals.contiguous()
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    with torch.cuda.device(flat.device), _timed("code_balance_backward"):
        check(_lib.lib().gsplat_hip_code_balance_backward(
            _balance_meta(flat, totals.shape[0], 1, 4), ptr(flat), ptr(counts), ptr(stats), ptr(totals), ptr(g[0]),
            ptr(g[1]), ptr(out), stream_of(flat)), "gsplat_hip_code_balance_backward")
    return out


@_balance_backward.register_fake
def _(g_loss, g_mean, logits, counts, stats, totals):
    return logits.new_empty(logits.shape)


def _balance_setup(ctx, inputs, output):
    _, counts, _, stats, totals = output
    ctx.mark_non_differentiable(counts, stats, totals)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(inputs[0], counts, stats, totals)


def _balance_grad(ctx, g_loss, _c, g_mean, *_):
    g = _balance_backward(g_loss, g_mean, *ctx.saved_tensors) if ctx.needs_input_grad[0] else None
    return g, None


_balance.register_autograd(_balance_grad, setup_context=_balance_setup)


# ---- checks


def _check_device(**tensors) -> None:
    names = [n for n, t in tensors.items() if t is not None]
    devices = {tensors[n].device for n in names}
    if len(devices) != 1:
        raise ValueError(f"{'/'.join(names)} must be on the same device")
    if devices.pop().type != "cuda":
        raise ValueError(f"{'/'.join(names)} must be ROCm device tensors (device type 'cuda')")


def _check_codes(codes: Tensor) -> None:
    if codes.dtype not in (torch.int32, torch.int64):
        raise ValueError("codes must be int32 or int64")


def _check_dtype(name: str, t: Tensor) -> None:
    if t.dtype not in _lib.DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16")


def _check_reverse(*tensors: Optional[Tensor]) -> None:
    """The operators have no forward derivative; torch would leave a dual input's tangent out."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("scenes in codes have gradients in reverse mode only, not in forward mode")


def _check_size(what: str, size: int, most: int) -> None:
    """The C ABI's limits, on sizes that its 32-bit fields have not cut."""
    if size > most:
        raise ValueError(f"at most {most} {what} are supported, not {size}")


def _check_given(name: str, t: Optional[Tensor], shape: Tuple[int, ...], dtype: torch.dtype, like: Tensor) -> None:
    """A backward operator's input, as its forward made it or as autograd passes it."""
    if t is None:
        return
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {str(dtype)[6:]}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} must be on the other inputs' device")


def _check_lookup(codes: Tensor, codebook: Tensor, scales: Optional[Tensor]) -> None:
    _check_codes(codes)
    _check_dtype("codebook", codebook)
    if codebook.ndim != 2 or 0 in codebook.shape:
        raise ValueError("codebook must have shape [K,D] with K and D at least 1")
    _check_size("codes", codebook.shape[0], _lib.MAX_CODES)
    _check_size("values per code", codebook.shape[1], _lib.MAX_CODE_WIDTH)
    if scales is not None:
        if scales.dtype != torch.float32:
            raise ValueError("scales must be float32")
        if scales.shape != codes.shape:
            raise ValueError("scales must match codes shape")
    _check_device(codes=codes, codebook=codebook, scales=scales)


def _check_logits(logits: Tensor) -> None:
    _check_dtype("logits", logits)
    if logits.ndim < 1 or logits.shape[-1] == 0:
        raise ValueError("logits must have a last axis of at least one code")


def _check_probs(logits: Tensor, codes: Optional[Tensor], top: int, temperature: float) -> None:
    _check_logits(logits)
    if codes is not None:
        _check_codes(codes)
        if codes.shape != logits.shape[:-1]:
            raise ValueError("codes must match logits shape without its last axis")
    most = min(_lib.MAX_TOP, logits.shape[-1])
    if not 0 <= top <= most:
        raise ValueError(f"top must lie in [0, {most}] (at most the number of codes, and {_lib.MAX_TOP})")
    if not (1e-30 <= temperature <= 1e30):
        raise ValueError("temperature must lie in [1e-30, 1e30]")
    _check_size("codes", logits.shape[-1], _lib.MAX_CODES)
    _check_device(logits=logits, codes=codes)


def _check_images(logits: Tensor) -> None:
    if logits.ndim not in (2, 3):
        raise ValueError("logits must have shape [G,K] or [B,G,K]")
    if logits.ndim == 3 and logits.shape[0] == 0:
        raise ValueError("at least one image is required (B >= 1)")
    _check_size("codes", logits.shape[-1], _lib.MAX_BALANCE_CODES)
    if logits.ndim == 3:
        _check_size("images", logits.shape[0], _lib.MAX_BALANCE_IMAGES)


def _check_balance(logits: Tensor, codes: Tensor) -> None:
    _check_logits(logits)
    _check_codes(codes)
    _check_images(logits)
    if codes.shape != logits.shape[:-1] and (codes.ndim != logits.ndim or codes.shape[:-1] != logits.shape[:-1]
                                             or codes.shape[-1] == 0):
        raise ValueError("codes must have the shape of logits without its last axis, or with choices per splat in its place")
    if codes.ndim == logits.ndim:
        _check_size("choices per splat", codes.shape[-1], _lib.MAX_CHOICES)
    _check_device(logits=logits, codes=codes)


# ---- the public calls


def lookup_codes(codes: Tensor, codebook: Tensor, scales: Optional[Tensor] = None, factor: float = 1.0) -> Tensor:
    """factor * scales[..., None] * codebook[codes]: attributes [..., D] of splats from their codes.

    codes [...] (-1: zeros), codebook [K,D], scales float32 of the codes' shape or None.  The result has
    the codebook's type.  Gradients flow to codebook and scales; a row of the codebook's gradient is the
    sum over the splats that name it, in an order that does not depend on the run."""
    out = _lib.host().lookup_codes(codes, codebook, scales, factor)
    if out is not None:
        return out
    _check_reverse(codebook, scales)
    _check_lookup(codes, codebook, scales)
    return _lookup(codes, codebook, scales, float(factor))


def code_log_probs(logits: Tensor, codes: Optional[Tensor] = None, top: int = 0, temperature: float = 1.0) -> CodeLogProbs:
    """Log probabilities under softmax(logits / temperature) over the codes (the last axis of logits).

    codes (the shape of logits without its last axis, or None): log_probs of those codes, 0 where a splat
    has none.  entropy: of every splat's distribution, in nats.  top > 0: the `top` likeliest codes, best
    first, and their log probabilities; among equal logits the lower code comes first, NaN ranks above
    everything.  A splat whose logits are all -inf has log probabilities of -inf, entropy 0 and no
    gradient.  Gradients flow from log_probs, entropy and top_log_probs to logits."""
    out = _lib.host().code_log_probs(logits, codes, top, temperature)
    if out is not None:
        return CodeLogProbs(*out)
    _check_reverse(logits)
    _check_probs(logits, codes, top, temperature)
    log_probs, entropy, top_log_probs, top_codes, _ = _probs(logits, codes, int(top), float(temperature))
    return CodeLogProbs(None if codes is None else log_probs, entropy, top_log_probs if top else None,
                        top_codes if top else None)


def code_balance(logits: Tensor, codes: Tensor) -> CodeBalance:
    """How evenly each image's splats use the codes.

    logits [G,K] or [B,G,K]; codes [G] or [B,G], or with several choices per splat [G,S] or [B,G,S].
    counts: choices of every code.  mean_probs: the mean of softmax(logits) over the splats that have a
    code.  loss = K * sum_k counts_k / (all choices) * mean_probs_k: 1 when both are even, larger the more
    they agree on a few codes; 0 for an image without any code.  Gradients flow from loss and mean_probs to
    logits (the counts are constants)."""
    out = _lib.host().code_balance(logits, codes)
    if out is not None:
        return CodeBalance(*out)
    _check_reverse(logits)
    _check_balance(logits, codes)
    loss, counts, mean_probs, _, _ = _balance(logits, codes)
    return CodeBalance(loss, counts, mean_probs)
