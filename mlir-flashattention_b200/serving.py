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

import ctypes
import struct
from typing import NamedTuple

import torch

from . import ATTN_BF16, ATTN_E4M3, ATTN_F16, ATTN_F32, VerifyError, _raise, lib

__all__ = ["AttnCachePlan", "AttnCacheAppend", "AttnRotary", "AttnTree", "CachePlan", "RotaryTable",
           "cache_plan", "cache_append", "rotary_table", "rotary", "fused_tree"]

_I, _Q, _P, _F = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
_DEVICE_POINTERS = 1  # flags: tensors here are known to be CUDA tensors


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


def _packer(cls):
    """struct.Struct with the C layout of a descriptor: one pack() fills it in a microsecond, which
    assigning forty ctypes fields does not."""
    code = {_I: "i", _Q: "q", _P: "P", _F: "f", _Q * 2: "2q", _Q * 3: "3q"}
    s = struct.Struct("@" + "".join(code[t] for _, t in cls._fields_) + "0q")
    assert s.size == ctypes.sizeof(cls)
    return s.pack


_pack_plan, _pack_append, _pack_rotary, _pack_tree = (
    _packer(c) for c in (AttnCachePlan, AttnCacheAppend, AttnRotary, AttnTree))

_CODES = {torch.float32: ATTN_F32, torch.bfloat16: ATTN_BF16, torch.float16: ATTN_F16,
          torch.float8_e4m3fn: ATTN_E4M3, torch.uint8: ATTN_E4M3}

_entries = {}


def _entry(name):
    fn = _entries.get(name)
    if fn is None:
        fn = getattr(lib(), name)
        fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_void_p]
        _entries[name] = fn
    return fn


def _call(name, desc, device):
    """Run an entry on the current stream of `device`."""
    index = device.index
    fn = _entry(name)
    if torch._C._cuda_getDevice() == index:
        rc = fn(desc, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(desc, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _raise(rc)


def _on_stream(stream):
    """The stream as torch's current one, so that what is allocated in a call belongs to it too."""
    return torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(stream))


def _need(ok, message):
    if not ok:
        raise VerifyError(message)


def _cuda(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise VerifyError(f"{name} must be a CUDA tensor on {device} (got {t.device})")


def _ints(t, name, shape, dtype=torch.int32):
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise VerifyError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of shape {list(shape)} "
                          f"(got {str(t.dtype)[6:]} {list(t.shape)})")


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise VerifyError(f"{what} has no backward pass: call it under torch.no_grad()")


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
        with _on_stream(stream):
            return cache_plan(lengths, targets, block_table, free_pages, free_count, page_size, tokens,
                              lengths_out=lengths_out, free_count_out=free_count_out, slots=slots,
                              positions=positions, starts=starts)
    _need(lengths.dim() == 1 and block_table.dim() == 2 and free_pages.dim() == 1,
          "lengths must be [B], block_table [B, W] and free_pages [num_pages]")
    B, W = block_table.shape
    shape, device = lengths.shape, lengths.device
    _need(device.type == "cuda", "lengths must be a CUDA tensor")
    _need(shape[0] == B, "lengths and block_table must have one row per request")
    _ints(lengths, "lengths", shape)
    _ints(targets, "targets", shape)
    _ints(free_pages, "free_pages", free_pages.shape)
    _ints(free_count, "free_count", (1,))
    _need(block_table.dtype == torch.int32 and (W <= 1 or block_table.stride(1) == 1),
          "block_table must be int32 with unit-stride columns")
    tokens = int(tokens)
    _need(tokens >= 0, "tokens must not be negative")
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    else:
        _ints(lengths_out, "lengths_out", shape)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    else:
        _ints(free_count_out, "free_count_out", (1,))
    if slots is None:
        slots = torch.empty(tokens, dtype=torch.int64, device=device)
    else:
        _ints(slots, "slots", (tokens,), torch.int64)
    if positions is None:
        positions = torch.empty(tokens, dtype=torch.int32, device=device)
    else:
        _ints(positions, "positions", (tokens,))
    if starts is None:
        starts = torch.empty(B + 1, dtype=torch.int32, device=device)
    else:
        _ints(starts, "starts", (B + 1,))
    _cuda(device, targets=targets, block_table=block_table, free_pages=free_pages, free_count=free_count,
          lengths_out=lengths_out, free_count_out=free_count_out, slots=slots, positions=positions, starts=starts)
    desc = _pack_plan(_DEVICE_POINTERS, int(page_size), B, W, free_pages.shape[0], tokens,
                      block_table.stride(0) if B > 1 else W, lengths.data_ptr(), targets.data_ptr(),
                      block_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), lengths_out.data_ptr(),
                      free_count_out.data_ptr(), starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), 0)
    _call("attn_cache_plan", desc, device)
    return CachePlan(slots, positions, starts, lengths_out, free_count_out)


# ------------------------------------------------------------------ cache writer
def _descale(value, name, heads, device):
    """(factor, pointer) of a descale: a number, or one f32 value per key head."""
    if isinstance(value, torch.Tensor):
        if value.dtype != torch.float32 or value.shape != (heads,) or not value.is_contiguous() or value.device != device:
            raise VerifyError(f"{name} must be a number or a contiguous f32 tensor of {heads} heads on {device}")
        return 1.0, value.data_ptr()
    return value, 0


def _check_cache(k_cache, v_cache, heads, dim, code, device):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[1] != heads or k_cache.shape[3] != dim:
        raise VerifyError(f"k_cache and v_cache must be [num_pages, {heads}, page_size, {dim}] "
                          f"(got {list(k_cache.shape)} and {list(v_cache.shape)})")
    if k_cache.dtype != v_cache.dtype or _CODES.get(k_cache.dtype, -1) not in (code, ATTN_E4M3):
        raise VerifyError(f"k_cache and v_cache must share one type: that of the keys, or float8_e4m3fn "
                          f"(got {k_cache.dtype} and {v_cache.dtype})")
    if k_cache.device != device or v_cache.device != device:
        raise VerifyError(f"k_cache and v_cache must be CUDA tensors on {device}")
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise VerifyError("the cache's head_dim must be unit-stride")
    return ks, vs


def cache_append(k, v, k_cache, v_cache, slots, *, rows=None, k_descale=1.0, v_descale=1.0, stream=None):
    """Write rows of ``k`` and ``v`` [T, Hkv, D] (bf16 or f16) to their cache slots, in place.

    Row ``rows[i]`` (int32 [N]; row i itself when None) goes to slot ``slots[i]`` (int64 [N], as
    :func:`cache_plan` makes them); a slot of -1 takes nothing.  Slots must differ.  A float8_e4m3fn
    cache holds x / descale, saturated to +-448; a descale is a number or an f32 tensor [Hkv].
    """
    if stream is not None:
        with _on_stream(stream):
            return cache_append(k, v, k_cache, v_cache, slots, rows=rows, k_descale=k_descale, v_descale=v_descale)
    if k.dim() != 3 or k.shape != v.shape:
        raise VerifyError("k and v must both be [tokens, heads, head_dim]")
    T, H, D = k.shape
    device, code = k.device, _CODES.get(k.dtype, -1)
    if device.type != "cuda" or v.device != device:
        raise VerifyError("k and v must be CUDA tensors on one device")
    if v.dtype != k.dtype or code not in (ATTN_BF16, ATTN_F16):
        raise VerifyError("k and v must both be bfloat16 or both float16")
    a, b = k.stride(), v.stride()
    if a[2] != 1 or b[2] != 1:
        raise VerifyError("head_dim must be unit-stride")
    ks, vs = _check_cache(k_cache, v_cache, H, D, code, device)
    n = slots.shape[0] if slots.dim() else 0
    _ints(slots, "slots", (n,), torch.int64)
    if rows is not None:
        _ints(rows, "rows", (n,))
    _cuda(device, slots=slots, rows=rows)
    _no_grad("cache_append", k, v)
    kd, kp = _descale(k_descale, "k_descale", H, device)
    vd, vp = _descale(v_descale, "v_descale", H, device)
    desc = _pack_append(_DEVICE_POINTERS, code, _CODES[k_cache.dtype], k_cache.shape[2], n, T, H, D, k_cache.shape[0],
                        a[0], a[1], b[0], b[1], *ks[:3], *vs[:3], k.data_ptr(), v.data_ptr(), k_cache.data_ptr(),
                        v_cache.data_ptr(), slots.data_ptr(), rows.data_ptr() if rows is not None else 0, kp, vp, kd,
                        vd, 0)
    _call("attn_cache_append", desc, device)


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


def _heads_strides(x, name, device, dtype):
    """(B, H, N, D, strides of batch, head, token) of [T, H, D] or [B, H, N, D]."""
    if x.device != device or x.dtype != dtype:
        raise VerifyError(f"{name} must be a {str(dtype)[6:]} tensor on {device}")
    s, n = x.stride(), x.shape
    if len(n) == 4:
        r = n[0], n[1], n[2], n[3], (s[0], s[1], s[2])
    elif len(n) == 3:
        r = 1, n[1], n[0], n[2], (0, s[1], s[0])
    else:
        raise VerifyError(f"{name} must be [tokens, heads, head_dim] or [batch, heads, tokens, head_dim]")
    if s[-1] != 1:
        raise VerifyError(f"{name} head_dim must be unit-stride")
    return r


def _rotate(q, k, positions, freqs, axes, neighbours, inverse, outs=(None, None)):
    first = q if q is not None else k
    device, dtype = first.device, first.dtype
    code = _CODES.get(dtype, -1)
    if device.type != "cuda":
        raise VerifyError("Q and K must be CUDA tensors")
    if code not in (ATTN_F32, ATTN_BF16, ATTN_F16):
        raise VerifyError(f"rotary takes float32, bfloat16 or float16 (got {dtype})")
    B, Hq, N, D, qs = _heads_strides(first, "Q", device, dtype)
    Hk, ks, q_out, k_out = 0, (0, 0, 0), outs[0], outs[1]
    if k is not None:
        b2, Hk, n2, d2, ks = _heads_strides(k, "K", device, dtype)
        if (b2, n2, d2) != (B, N, D) or k.dim() != first.dim():
            raise VerifyError("Q and K must have the same tokens and head_dim")
        if k_out is None:
            k_out = torch.empty_like(k)
    if q is None:
        Hq, qs = 0, (0, 0, 0)
    elif q_out is None:
        q_out = torch.empty_like(q)
    half = freqs.shape[0] if freqs.dim() else 0
    if freqs.dtype != torch.float64 or freqs.shape != (half,) or not freqs.is_contiguous():
        raise VerifyError("freqs must be a contiguous float64 tensor [dim / 2]")
    if 2 * half > D:
        raise VerifyError(f"freqs turn {2 * half} values of a head_dim of {D}")
    if axes is not None:
        _ints(axes, "axes", (half,))
    p = positions
    if p.dtype not in (torch.int32, torch.int64):
        raise VerifyError("positions must be int32 or int64")
    if p.dim() == 1:
        p = p.unsqueeze(0)
    ps = p.stride()
    if p.dim() == 3 and first.dim() == 4 and p.shape[1:] == (B, N):
        pos_stride = ps
    elif p.dim() == 2 and p.shape[1] == N:
        pos_stride = (ps[0], 0, ps[1])
    else:
        raise VerifyError(f"positions must be [axes, {N}]" + (f" or [axes, {B}, {N}]" if first.dim() == 4 else "") +
                          f" (got {list(positions.shape)})")
    if p.shape[0] == 0:
        raise VerifyError("positions need an axis")
    _cuda(device, positions=p, freqs=freqs, axes=axes)
    zero = (0, 0, 0)
    qos = _heads_strides(q_out, "q output", device, dtype)[4] if q is not None else zero
    kos = _heads_strides(k_out, "k output", device, dtype)[4] if k is not None else zero
    desc = _pack_rotary(_DEVICE_POINTERS, code, p.dtype == torch.int64, p.shape[0], bool(neighbours), bool(inverse), B, N,
                        Hq, Hk, D, 2 * half, *qs, *ks, *qos, *kos, *pos_stride, q.data_ptr() if q is not None else 0,
                        k.data_ptr() if k is not None else 0, q_out.data_ptr() if q is not None else 0,
                        k_out.data_ptr() if k is not None else 0, p.data_ptr(), freqs.data_ptr(),
                        axes.data_ptr() if axes is not None else 0, 0)
    _call("attn_rotary", desc, device)
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """A turn; its gradient is the turn back, itself a turn (so differentiable again)."""

    @staticmethod
    def forward(ctx, q, k, positions, freqs, axes, neighbours, inverse):
        ctx.save_for_backward(positions, freqs, axes)
        ctx.how = neighbours, inverse
        ctx.set_materialize_grads(False)
        return _rotate(q, k, positions, freqs, axes, neighbours, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        positions, freqs, axes = ctx.saved_tensors
        neighbours, inverse = ctx.how
        gq, gk = (g if g is None or g.stride(-1) == 1 else g.contiguous() for g in (gq, gk))
        if gq is not None or gk is not None:
            gq, gk = _apply_rotary(gq, gk, positions, freqs, axes, neighbours, not inverse)
        return gq, gk, None, None, None, None, None


def _apply_rotary(q, k, positions, freqs, axes, neighbours, inverse):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k)):
        return _Rotary.apply(q, k, positions, freqs, axes, neighbours, inverse)
    return _rotate(q, k, positions, freqs, axes, neighbours, inverse)


def rotary(q, k, positions, freqs, axes=None, *, neighbours=False, inverse=False, stream=None):
    """Turn Q and K by their positions: pair i of the first 2 len(freqs) values of a head by
    ``positions[axes[i]] * freqs[i]`` radians, (x, y) -> (x cos - y sin, x sin + y cos).

    Q and K are [tokens, heads, head_dim] or [batch, heads, tokens, head_dim] in f32, bf16 or f16;
    either may be None.  ``positions`` is int32 or int64 [axes, tokens] (for rank 4 also
    [axes, batch, tokens]; [tokens] for a single axis).  ``freqs`` [dim/2] float64 and ``axes``
    [dim/2] int32 come from :func:`rotary_table` (a whole table may stand in their place).  Pairs are
    (i, i + dim/2), or (2i, 2i + 1) with ``neighbours``; values behind them are copied.  ``inverse``
    turns back.  Returns the turned (q, k); differentiable in both.
    """
    if isinstance(freqs, RotaryTable):
        freqs, axes, neighbours = freqs
    if q is None and k is None:
        raise VerifyError("rotary needs Q or K")
    if stream is not None:
        with _on_stream(stream):
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
    tokens of a request (default T).  A row that sees nothing gets O = 0 and LSE = -inf; rows past
    ``starts[B]`` are left as they were.  ``lse`` (f32 [T, Hq]) receives the natural-log sums.
    """
    if stream is not None:
        with _on_stream(stream):
            return fused_tree(q, k_new, v_new, k_cache, v_cache, block_table, lengths, starts, scale, mask=mask,
                              max_new=max_new, output=output, lse=lse, k_descale=k_descale, v_descale=v_descale)
    if q.dim() != 3 or k_new.dim() != 3 or k_new.shape != v_new.shape:
        raise VerifyError("Q, K and V must be [tokens, heads, head_dim]")
    T, Hq, D = q.shape
    Tk, H, Dk = k_new.shape
    if Tk != T:
        raise VerifyError("K seq_len must equal Q seq_len")
    if Dk != D:
        raise VerifyError("K head_dim must equal Q head_dim")
    device, code = q.device, _CODES.get(q.dtype, -1)
    if device.type != "cuda" or k_new.device != device or v_new.device != device:
        raise VerifyError("Q, K and V must be CUDA tensors on one device")
    if code not in (ATTN_BF16, ATTN_F16) or k_new.dtype != q.dtype or v_new.dtype != q.dtype:
        raise VerifyError("Q, K and V must share one element type, bfloat16 or float16")
    qs, ns, ws = q.stride(), k_new.stride(), v_new.stride()
    if qs[2] != 1 or ns[2] != 1 or ws[2] != 1:
        raise VerifyError("head_dim must be unit-stride")
    ks, vs = _check_cache(k_cache, v_cache, H, D, code, device)
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise VerifyError("block_table must be int32 [B, W] with unit-stride columns")
    B, W = block_table.shape
    _ints(lengths, "lengths", (B,))
    _ints(starts, "starts", (B + 1,))
    max_new = T if max_new is None else int(max_new)
    mask_stride = 0
    if mask is not None:
        if (mask.dim() != 2 or mask.dtype not in (torch.bool, torch.uint8) or mask.shape[0] != T or
                mask.shape[1] < max_new or (mask.shape[1] > 1 and mask.stride(1) != 1)):
            raise VerifyError(f"mask must be bool [{T}, at least max_new = {max_new}] with unit-stride columns")
        mask_stride = mask.stride(0) if T > 1 else mask.shape[1]
    if output is None:
        output = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    elif output.shape != q.shape or output.dtype != q.dtype or output.stride(2) != 1:
        raise VerifyError("output must have Q's shape and type, head_dim unit-stride")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (T, Hq) or not lse.is_contiguous()):
        raise VerifyError("lse must be a contiguous f32 tensor [tokens, heads]")
    _cuda(device, block_table=block_table, lengths=lengths, starts=starts, mask=mask, output=output, lse=lse)
    _no_grad("fused_tree", q, k_new, v_new)
    kd, kp = _descale(k_descale, "k_descale", H, device)
    vd, vp = _descale(v_descale, "v_descale", H, device)
    os = output.stride()
    desc = _pack_tree(_DEVICE_POINTERS, code, _CODES[k_cache.dtype], k_cache.shape[2], B, T, Hq, H, D, W, k_cache.shape[0],
                      max_new, qs[0], qs[1], ns[0], ns[1], ws[0], ws[1], os[0], os[1], *ks[:3], *vs[:3],
                      block_table.stride(0) if B > 1 else W, mask_stride, q.data_ptr(), k_new.data_ptr(),
                      v_new.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), output.data_ptr(),
                      lse.data_ptr() if lse is not None else 0, block_table.data_ptr(), lengths.data_ptr(),
                      starts.data_ptr(), mask.data_ptr() if mask is not None else 0, kp, vp, scale, kd, vd, 0)
    _call("attn_tree_fwd", desc, device)
    return output
