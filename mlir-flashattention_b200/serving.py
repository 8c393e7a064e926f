"""Serving: a paged key/value cache, what fills it, and the attention that reads it.

``fused`` attends over whole Q, K and V.  A model served token by token keeps the keys and values
of the tokens seen so far in pages and attends from a few new tokens at a time:

* :func:`cache_plan` grows and shrinks the requests' page lists on the GPU and gives every new
  token its position and cache slot;
* :func:`rotary` turns Q and K by positions with one or several axes (differentiable);
* :func:`fused_tree` attends from each request's new tokens (a decoded token, a drafted tree or a
  chunk of a prompt) over its cached tokens and over each other;
* :func:`cache_append` writes the accepted tokens' keys and values to their slots.

The cache is a pair of tensors ``[num_pages, Hkv, page_size, D]`` (any strides with unit head_dim
stride, so a ``[num_pages, page_size, Hkv, D]`` layout is a transposed view).  Every call is one
entry of ``include/attn_rt.h``: asynchronous, without a look at device data.  Wrong shapes and types
raise :class:`VerifyError` here; what only the device can see (a page or slot out of range, a pool
run empty) is recorded in the runtime's status word, which ``check_status`` raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
from typing import NamedTuple

import torch

from . import _HERE, LIB_PATH, AttentionError, VerifyError, lib

__all__ = ["AttnCachePlan", "AttnCacheAppend", "AttnRotary", "AttnTree", "CachePlan", "RotaryTable",
           "cache_plan", "cache_append", "rotary_table", "rotary", "fused_tree"]

_I, _Q, _P, _F = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float


class AttnCachePlan(ctypes.Structure):
    _fields_ = [("flags", _I), ("page_size", _I), ("B", _Q), ("W", _Q), ("num_pages", _Q), ("tokens", _Q),
                ("table_stride", _Q), ("lengths", _P), ("targets", _P), ("block_table", _P), ("free_pages", _P),
                ("free_count", _P), ("lengths_out", _P), ("free_count_out", _P), ("starts", _P), ("positions", _P),
                ("slots", _P), ("status", _P)]


class AttnCacheAppend(ctypes.Structure):
    _fields_ = [("flags", _I), ("dtype", _I), ("cache_dtype", _I), ("page_size", _I), ("N", _Q), ("T", _Q), ("Hkv", _Q),
                ("D", _Q), ("num_pages", _Q), ("k_stride", _Q * 2), ("v_stride", _Q * 2), ("k_cache_stride", _Q * 3),
                ("v_cache_stride", _Q * 3), ("k", _P), ("v", _P), ("k_cache", _P), ("v_cache", _P), ("slots", _P),
                ("rows", _P), ("k_descale_heads", _P), ("v_descale_heads", _P), ("k_descale", _F), ("v_descale", _F),
                ("status", _P)]


class AttnRotary(ctypes.Structure):
    _fields_ = [("flags", _I), ("dtype", _I), ("positions_64", _I), ("num_axes", _I), ("neighbours", _I), ("inverse", _I),
                ("B", _Q), ("N", _Q), ("Hq", _Q), ("Hk", _Q), ("D", _Q), ("R", _Q), ("q_stride", _Q * 3),
                ("k_stride", _Q * 3), ("qo_stride", _Q * 3), ("ko_stride", _Q * 3), ("pos_stride", _Q * 3), ("q", _P),
                ("k", _P), ("qo", _P), ("ko", _P), ("positions", _P), ("freqs", _P), ("axes", _P), ("status", _P)]


class AttnTree(ctypes.Structure):
    _fields_ = [("flags", _I), ("dtype", _I), ("cache_dtype", _I), ("page_size", _I), ("B", _Q), ("T", _Q), ("Hq", _Q),
                ("Hkv", _Q), ("D", _Q), ("W", _Q), ("num_pages", _Q), ("max_new", _Q), ("q_stride", _Q * 2),
                ("k_stride", _Q * 2), ("v_stride", _Q * 2), ("o_stride", _Q * 2), ("k_cache_stride", _Q * 3),
                ("v_cache_stride", _Q * 3), ("table_stride", _Q), ("mask_stride", _Q), ("q", _P), ("k_new", _P),
                ("v_new", _P), ("k_cache", _P), ("v_cache", _P), ("o", _P), ("lse", _P), ("block_table", _P),
                ("lengths", _P), ("starts", _P), ("mask", _P), ("k_descale_heads", _P), ("v_descale_heads", _P),
                ("scale", _F), ("k_descale", _F), ("v_descale", _F), ("status", _P)]


_module = None


def _native():
    """The calls on torch tensors (_serving.so: checks, descriptors, the current stream)."""
    global _module
    if _module is None:
        import importlib.util  # noqa: PLC0415
        lib()
        path = os.path.join(_HERE, "_serving.so")
        if not os.path.exists(path):
            raise RuntimeError(f"_serving.so not found at {path}; build it with __graft_entry__.build()")
        spec = importlib.util.spec_from_file_location("_serving", path)
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        m.setup(LIB_PATH, VerifyError, AttentionError)
        _module = m
    return _module


def _on_stream(stream, operand):
    """The stream (a torch stream or a raw handle, of the operand's device) as torch's current one, so that what is
    allocated in a call belongs to it too."""
    device = getattr(operand, "device", None)
    if device is None or device.type != "cuda":
        return contextlib.nullcontext()  # which the call refuses
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(stream, device=device)
    _need(stream.device == device, f"stream must belong to {device} (got one of {stream.device})")
    return torch.cuda.stream(stream)


def _need(ok, message):
    if not ok:
        raise VerifyError(message)


# ------------------------------------------------------------------ page planner
class CachePlan(NamedTuple):
    """What :func:`cache_plan` says of a step."""
    slots: torch.Tensor       # [tokens] int64: cache slot of each new token, -1 past the last
    positions: torch.Tensor   # [tokens] int32: its position in its request, 0 past the last
    starts: torch.Tensor      # [B + 1] int32: new tokens of the requests before each
    lengths: torch.Tensor     # [B] int32: tokens then held
    free_count: torch.Tensor  # [1] int32: pages then free


def cache_plan(lengths, targets, block_table, free_pages, free_count, page_size, tokens, *, lengths_out=None,
               free_count_out=None, slots=None, positions=None, starts=None, stream=None) -> CachePlan:
    """Grow or shrink each request from ``lengths[b]`` to ``targets[b]`` tokens (both [B] int32).

    ``block_table`` [B, W] int32 lists each request's pages and ``free_pages`` [num_pages] int32 is a
    stack of the free ones with ``free_count`` [1] int32 entries; both are written in place.  Pages of
    shrinking requests (a finished one shrinks to 0) are pushed, request by request in page order; then
    growing requests pop theirs in the same order.  ``tokens`` is the length of ``slots`` and
    ``positions``: at least the new tokens in all, or a padded number.

    ``lengths_out`` and ``free_count_out`` may be the inputs themselves (in place, as in a captured
    decode loop); by default they are new.  The call is all or nothing: where pages, table columns or
    ``tokens`` do not suffice, nothing changes, starts are 0, slots are -1 and the status word holds
    ATTN_ERR_CAPACITY (ATTN_ERR_INVALID for a length that cannot be).
    """
    if stream is not None:
        with _on_stream(stream, lengths):
            return cache_plan(lengths, targets, block_table, free_pages, free_count, page_size, tokens,
                              lengths_out=lengths_out, free_count_out=free_count_out, slots=slots,
                              positions=positions, starts=starts)
    return CachePlan._make((_module or _native()).plan(lengths, targets, block_table, free_pages, free_count, page_size,
                                                       tokens, lengths_out, free_count_out, slots, positions, starts))


# ------------------------------------------------------------------ cache writer
def cache_append(k, v, k_cache, v_cache, slots, *, rows=None, k_descale=1.0, v_descale=1.0, stream=None):
    """Write rows of ``k`` and ``v`` [T, Hkv, D] (bf16 or f16) to their cache slots, in place.

    Row ``rows[i]`` (int32 [N]; row i itself when None) goes to slot ``slots[i]`` (int64 [N], as
    :func:`cache_plan` makes them); a slot of -1 takes nothing.  Slots must differ.  A float8_e4m3fn
    cache holds x / descale, saturated to +-448; a descale is a number or an f32 tensor [Hkv].  Operands
    that require a gradient, or carry a forward-mode tangent, are refused.
    """
    if stream is not None:
        with _on_stream(stream, k):
            return cache_append(k, v, k_cache, v_cache, slots, rows=rows, k_descale=k_descale, v_descale=v_descale)
    (_module or _native()).append(k, v, k_cache, v_cache, slots, rows, k_descale, v_descale)


# ------------------------------------------------------------------ rotary positions
class RotaryTable(NamedTuple):
    """Frequencies of a rotary embedding, laid out once."""
    freqs: torch.Tensor  # [dim / 2] float64: radians per position of each pair
    axes: torch.Tensor   # [dim / 2] int32: the axis whose position turns it
    neighbours: bool     # pairs (2i, 2i + 1) instead of (i, i + dim / 2)


def rotary_table(dim, sections=None, base=10000.0, *, interleaved=False, neighbours=False, device="cuda"):
    """The table of a rotary embedding over the first ``dim`` values of a head: pair i turns by
    base^(-2i/dim) radians a position.  ``sections`` gives the number of pairs of each axis (time,
    height, width), in all dim/2; the pairs belong to the axes one section after another, or in turn
    (``interleaved``) while an axis has pairs left.  None is a single axis."""
    half = dim // 2
    sections = [half] if sections is None else [int(n) for n in sections]
    _need(dim > 0 and dim % 2 == 0, "dim must be positive and even")
    _need(min(sections) >= 0 and sum(sections) == half, f"sections must sum to dim / 2 = {half} (got {sections})")
    if interleaved:
        axes = [a for turn in range(max(sections)) for a, n in enumerate(sections) if turn < n]
    else:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    freqs = float(base) ** (-torch.arange(half, dtype=torch.float64) * 2 / dim)
    return RotaryTable(freqs.to(device), torch.tensor(axes, dtype=torch.int32, device=device), bool(neighbours))


class _Rotary(torch.autograd.Function):
    """A turn; its gradient is the turn back, itself a turn (so differentiable again)."""

    @staticmethod
    def forward(ctx, q, k, positions, freqs, axes, neighbours, inverse):
        ctx.save_for_backward(positions, freqs, axes)
        ctx.save_for_forward(positions, freqs, axes)
        ctx.how = neighbours, inverse
        ctx.set_materialize_grads(False)
        out = (_module or _native()).rotate(q, k, positions, freqs, axes, neighbours, inverse)
        ctx.form = [None if x is None else (x.shape, x.dtype, x.device) for x in out]
        return out

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        """Tangents turn as the values do; an operand without one has the tangent 0."""
        positions, freqs, axes = ctx.saved_tensors
        tq, tk = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (tq, tk))
        turned = _apply_rotary(tq, tk, positions, freqs, axes, *ctx.how)
        return tuple(torch.zeros(f[0], dtype=f[1], device=f[2]) if t is None and f else t
                     for t, f in zip(turned, ctx.form))

    @staticmethod
    def backward(ctx, gq, gk):
        positions, freqs, axes = ctx.saved_tensors
        neighbours, inverse = ctx.how
        gq, gk = (g if g is None or g.stride(-1) == 1 else g.contiguous() for g in (gq, gk))
        if gq is not None or gk is not None:
            gq, gk = _apply_rotary(gq, gk, positions, freqs, axes, neighbours, not inverse)
        return gq, gk, None, None, None, None, None


def _apply_rotary(q, k, positions, freqs, axes, neighbours, inverse):
    native = _module or _native()
    if (((q is not None and q.requires_grad) or (k is not None and k.requires_grad)) and torch.is_grad_enabled()) \
            or native.dual(q, k):
        return _Rotary.apply(q, k, positions, freqs, axes, neighbours, inverse)
    return native.rotate(q, k, positions, freqs, axes, neighbours, inverse)


def rotary(q, k, positions, freqs, axes=None, *, neighbours=False, inverse=False, stream=None):
    """Turn Q and K by their positions: pair i of the first 2 len(freqs) values of a head by
    ``positions[axes[i]] * freqs[i]`` radians, (x, y) -> (x cos - y sin, x sin + y cos).

    Q and K are [tokens, heads, head_dim] or [batch, heads, tokens, head_dim] in f32, bf16 or f16;
    either may be None.  ``positions`` is int32 or int64 [axes, tokens] (for rank 4 also
    [axes, batch, tokens]; [tokens] for a single axis).  ``freqs`` [dim/2] float64 and ``axes``
    [dim/2] int32 come from :func:`rotary_table` (a whole table may stand in their place).  Pairs are
    (i, i + dim/2), or (2i, 2i + 1) with ``neighbours``; values behind them are copied.  ``inverse``
    turns back.  Returns the turned (q, k); differentiable in both, backward and by forward-mode tangents
    (``torch.autograd.forward_ad``; the transforms of ``torch.func`` are refused).
    """
    if isinstance(freqs, RotaryTable):
        freqs, axes, neighbours = freqs
    if stream is not None:
        with _on_stream(stream, k if q is None else q):
            return _apply_rotary(q, k, positions, freqs, axes, neighbours, inverse)
    return _apply_rotary(q, k, positions, freqs, axes, neighbours, inverse)


# ------------------------------------------------------------------ attention over the cache
def fused_tree(q, k_new, v_new, k_cache, v_cache, block_table, lengths, starts, scale, *, mask=None, max_new=None,
               output=None, lse=None, k_descale=1.0, v_descale=1.0, stream=None):
    """Attention of each request's new tokens over its cached tokens and over each other:
    ``O = softmax(scale * Q·Kᵀ)·V`` over the keys a token sees.

    q [T, Hq, D], k_new and v_new [T, Hkv, D] (bf16 or f16; Hq a multiple of Hkv) hold the new tokens
    of all requests one after another: rows ``starts[b]`` to ``starts[b + 1]`` (int32 [B + 1]) are
    request b's.  Each sees all ``lengths[b]`` (int32 [B]) cached tokens, whose pages
    ``block_table[b]`` lists in k_cache and v_cache [num_pages, Hkv, page_size, D] (q's type, or
    float8_e4m3fn with descales: numbers or f32 tensors [Hkv]).  The new tokens need not be in the
    cache: :func:`cache_append` can write the accepted ones afterwards.

    ``mask`` (bool or uint8 [T, >= max_new], True = masked) says which new tokens of its request a
    row does not see: all but itself and its ancestors for a drafted tree.  Without a mask a row sees
    itself and those before it: a decoded token, or a chunk of a prompt.  ``max_new`` bounds the new
    tokens of a request (default T) and chooses the kernel for the whole call, so give it: 1 for a
    step of decoded tokens, which without it would run as a call for many rows.  A row that sees
    nothing gets O = 0 and LSE = -inf, one whose scores are no numbers or all -inf an O that is none;
    rows past ``starts[B]`` are left as they were.  ``lse`` (f32 [T, Hq]) receives the natural-log
    sums.  ``output`` may be q itself, but must not overlap the other operands.  There is no backward
    pass: operands that require a gradient, or carry a forward-mode tangent, are refused.
    """
    if stream is not None:
        with _on_stream(stream, q):
            return fused_tree(q, k_new, v_new, k_cache, v_cache, block_table, lengths, starts, scale, mask=mask,
                              max_new=max_new, output=output, lse=lse, k_descale=k_descale, v_descale=v_descale)
    return (_module or _native()).tree(q, k_new, v_new, k_cache, v_cache, block_table, lengths, starts, scale, mask, max_new,
                                       output, lse, k_descale, v_descale)
