"""The paged key/value cache of a served model: append, attention, eviction.

Keys and values of all sequences live in pages, ``k_pages`` and ``v_pages``
(num_pages, Hkv, page_size, 64), bfloat16 or float32, page_size a power of two
from 16 to 256. ``table`` (B, max_pages) int32 names each sequence's pages and
``lens`` (B) int32 its cached slots: slot ``s`` is row ``s % page_size`` of page
``table[b, s // page_size]``. A decode step is

    q = cache_append(qkv, k_pages, v_pages, table, lens, gain_q, gain_k, rotary=rot)
    o = paged_attention(q, k_pages, v_pages, table, lens + T, sink, n=16, c=8.0)

and, for a cache that must not grow, ``paged_attention(..., scores=scores)``
accumulates the attention weight every slot received and ``cache_evict`` keeps
the slots that received most. Everything runs on the current stream without
host synchronisation, so a step can be captured in a CUDA graph; page numbers,
lengths and positions are read on the device, and one outside its range is
skipped and raises the device error word (``algx._lib.device_error()``) instead
of being followed. No gradients: these are serving operators (the training path
is ``algx.kernels.flash``). The reference has no cache; the formulas are its
QK norm (qk_norm.py:29-43), rotation (algebraic.py:172-179) and attention
weights (algebraic.py:186-216, standard.py:24-38).
"""

from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from .. import _lib as L

_CODE = {torch.bfloat16: L.ALGX_BF16, torch.float32: L.ALGX_F32}
_SIZES = frozenset((16, 32, 64, 128, 256))
_I32, _F32 = torch.int32, torch.float32


# A decode step makes these calls once per layer on small tensors, where the
# host's time is the call's: the checks read each attribute once.
def _check_cache(k_pages, v_pages, table, lens):
    """Shapes and dtypes of a paged cache; returns (num_pages, Hkv, page_size, B, max_pages, dtype code)."""
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != dtype:
        raise ValueError("k_pages and v_pages must both have shape (num_pages, heads, page_size, 64) and one dtype")
    num, heads, size, D = shape
    if D != 64:
        raise ValueError(f"algx paged cache supports head_dim 64, got {D}")
    code = _CODE.get(dtype)
    if code is None:
        raise ValueError("paged cache must be bfloat16 or float32")
    if size not in _SIZES:
        raise ValueError(f"page_size must be a power of two from 16 to 256, got {size}")
    if num < 1 or heads < 1:
        raise ValueError("paged cache has no pages or no heads")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous")
    tshape = table.shape
    if len(tshape) != 2 or lens.shape != tshape[:1] or tshape[1] < 1:
        raise ValueError("table must have shape (B, max_pages) and lens (B,)")
    if table.dtype != _I32 or lens.dtype != _I32:
        raise ValueError("table and lens must be int32")
    return num, heads, size, tshape[0], tshape[1], code


def _check_state(name, t, shape, dtype):
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of shape {shape}")


def _same_device(ref, *tensors):
    dev = ref.get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            L.require_cuda(ref, t)
            raise ValueError(f"tensors on {ref.device} and {t.device} in one call")
    if dev < 0:
        L.require_cuda(ref)


def _ready(t):
    """``t`` contiguous at a 16-byte boundary, as the kernels load it (a copy where it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() & 15 == 0 else t.clone()


def _per_sequence(name, t, B):
    if t.shape != (B,) or t.dtype != _I32:
        raise ValueError(f"{name} must be int32 of shape ({B},)")
    return t.contiguous()


def cache_append(qkv, k_pages, v_pages, table, lens, gain_q=None, gain_k=None, *, rotary=None, positions=None,
                 counts=None, slot_positions=None, eps: float = 1e-5):
    """Put the keys and values of T new tokens per sequence into the cache; returns their queries (B, T, Hq, 64).

    ``qkv`` (B, T, Hq + 2 Hkv, 64) holds the [q | k | v] heads of each token
    (the model's packed (B, T, 3, H, 64) projection is its (B, T, 3 H, 64) view).
    ``lens``: slots held before the call; token t goes to slot ``lens[b] + t``
    and the call changes no length. ``gain_q``, ``gain_k`` (64,) float32 apply
    the QK RMS norm, ``rotary`` = (cos, sin), each (rows, 32) float32, the
    rotation at position ``positions[b] + t`` (default: the slot). Norm and
    rotation are evaluated in float32 and rounded once. ``counts`` (B,) int32:
    tokens beyond it are padding, stored nowhere, their queries zero.
    ``slot_positions`` (B, Hkv, max_pages * page_size) int32 receives the new
    slots' positions, which ``cache_evict`` reads.
    """
    num, Hkv, size, B, maxp, code = _check_cache(k_pages, v_pages, table, lens)
    shape = qkv.shape
    if len(shape) != 4 or shape[0] != B or shape[3] != 64 or shape[2] < 2 * Hkv:
        raise ValueError(f"qkv must have shape ({B}, T, Hq + {2 * Hkv}, 64), got {tuple(shape)}")
    if qkv.dtype != k_pages.dtype:
        raise ValueError(f"qkv ({qkv.dtype}) and the cache ({k_pages.dtype}) must share one dtype")
    if (gain_q is None) != (gain_k is None):
        raise ValueError("give both gain_q and gain_k or neither")
    if eps <= 0:
        raise ValueError("eps must be positive")
    cos = sin = None
    rows = 0
    if gain_q is not None:
        for g in (gain_q, gain_k):
            if g.shape != (64,) or g.dtype != _F32:
                raise ValueError("gains must be float32 of shape (64,)")
        gain_q, gain_k = _ready(gain_q), _ready(gain_k)
    if rotary is not None:
        cos, sin = rotary
        rshape = cos.shape
        if len(rshape) != 2 or rshape[1] != 32 or sin.shape != rshape or cos.dtype != _F32 or sin.dtype != _F32 \
                or rshape[0] < 1:
            raise ValueError("rotary tables must both be float32 of shape (rows, 32)")
        cos, sin = _ready(cos), _ready(sin)
        rows = rshape[0]
    if positions is not None:
        positions = _per_sequence("positions", positions, B)
    if counts is not None:
        counts = _per_sequence("counts", counts, B)
    if slot_positions is not None:
        _check_state("slot_positions", slot_positions, (B, Hkv, maxp * size), _I32)
    _same_device(qkv, k_pages, v_pages, table, lens, gain_q, gain_k, cos, sin, positions, counts, slot_positions)
    qkv, table, lens = _ready(qkv), table.contiguous(), lens.contiguous()
    T, Hq = shape[1], shape[2] - 2 * Hkv
    q = qkv.new_empty((B, T, Hq, 64))
    L.check(L.lib().algx_cache_append(
        qkv.data_ptr(), L.ptr(gain_q), L.ptr(gain_k), L.ptr(cos), L.ptr(sin), rows, table.data_ptr(), lens.data_ptr(),
        L.ptr(positions), L.ptr(counts), q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), L.ptr(slot_positions),
        B, T, Hq, Hkv, num, size, maxp, 64, code, eps, L.stream_of(qkv)), "algx_cache_append")
    return q


@functools.lru_cache(maxsize=256)
def paged_config(kind: str, n: int, c: float, window: Optional[int], first: int) -> L.PagedConfig:
    """The C ABI's configuration of one kind of paged attention (checked, cached by value)."""
    if kind not in ("asinh", "softmax"):
        raise ValueError(f"unknown attention kernel: {kind}")
    if kind == "asinh" and (n < 2 or n & (n - 1)):
        raise ValueError("asinh kernel needs n to be a power of two")
    if kind == "asinh" and (not math.isfinite(c) or c <= 0):
        raise ValueError("asinh scale c must be positive and finite")
    if window is not None and not 1 <= window < 2 ** 31:
        raise ValueError("window must be positive")
    if not 0 <= first < 2 ** 31:
        raise ValueError("first must not be negative")
    unit = float(c) if kind == "asinh" else 1.0
    return L.PagedConfig(L.ALGX_ATTN_ASINH if kind == "asinh" else L.ALGX_ATTN_SOFTMAX,
                         int(n) if kind == "asinh" else 2, window or 0, first, 1.0 / (8.0 * unit), 1.0 / unit)


@functools.lru_cache(maxsize=4096)
def _attn_workspace(*sizes) -> int:
    """``algx_paged_attn_workspace_size``, a function of its arguments alone."""
    return max(L.lib().algx_paged_attn_workspace_size(*sizes), 1)


def paged_attention(q, k_pages, v_pages, table, lens, sink_logit=None, *, kind: str = "softmax", n: int = 16,
                    c: float = 16.0, window: Optional[int] = None, first: int = 0, scores=None, scores_out=None):
    """Attention of the T newest tokens of every sequence over its cached slots; returns o (B, T, Hq, 64).

    ``q`` (B, T, Hq, 64) in the cache's dtype, Hq a multiple of the cache's
    heads; ``lens`` (B,) counts the cached slots, the T new ones included, and
    query t sees the slots up to its own, ``lens[b] - T + t``. ``window``: only
    the newest ``window`` slots up to its own stay visible, and the ``first``
    first ones of the sequence. ``kind``, ``n``, ``c`` and ``sink_logit``
    (broadcastable to (Hq,)) are those of
    ``algx.kernels.flash.flash_attention``; the asinh kind is evaluated against a
    running maximum, so any score range is safe. A query that sees nothing gives
    zeros.

    ``scores`` (B, Hkv, max_pages * page_size) float32: the weight every slot
    has received; the call adds its own normalised weights, summed over the
    queries of each kv head, into ``scores_out`` (default: ``scores`` itself) and
    returns ``(o, scores_out)``. The T new slots start from zero, slots beyond
    ``lens`` are set to zero.
    """
    num, Hkv, size, B, maxp, code = _check_cache(k_pages, v_pages, table, lens)
    shape = q.shape
    if len(shape) != 4 or shape[0] != B or shape[3] != 64 or shape[2] < 1 or shape[2] % Hkv:
        raise ValueError(f"q must have shape ({B}, T, Hq, 64) with Hq a multiple of {Hkv}, got {tuple(shape)}")
    if q.dtype != k_pages.dtype:
        raise ValueError(f"q ({q.dtype}) and the cache ({k_pages.dtype}) must share one dtype")
    cfg = paged_config(kind, n, c, window, first)
    T, Hq = shape[1], shape[2]
    sink = None
    if sink_logit is not None:
        sink = sink_logit
        if not torch.is_tensor(sink) or sink.dtype != _F32 or sink.shape != (Hq,) or sink.device != q.device:
            sink = torch.as_tensor(sink, dtype=_F32, device=q.device)
            sink = torch.broadcast_to(sink.reshape(-1), (Hq,))
        sink = sink.contiguous()
    if scores is not None:
        scores_out = scores if scores_out is None else scores_out
        _check_state("scores", scores, (B, Hkv, maxp * size), _F32)
        _check_state("scores_out", scores_out, (B, Hkv, maxp * size), _F32)
    elif scores_out is not None:
        raise ValueError("scores_out without scores")
    _same_device(q, k_pages, v_pages, table, lens, scores, scores_out)
    q, table, lens = _ready(q), table.contiguous(), lens.contiguous()
    o = torch.empty_like(q)
    nbytes = _attn_workspace(B, T, Hq, Hkv, size, maxp, scores is not None, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    L.check(L.lib().algx_paged_attn(
        cfg, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lens.data_ptr(), L.ptr(sink),
        L.ptr(scores), L.ptr(scores_out), o.data_ptr(), B, T, Hq, Hkv, num, size, maxp, 64, code, ws.data_ptr(),
        nbytes, L.stream_of(q)), "algx_paged_attn")
    return o if scores is None else (o, scores_out)


@functools.lru_cache(maxsize=4096)
def _evict_workspace(*sizes) -> int:
    return max(L.lib().algx_cache_evict_workspace_size(*sizes), 1)


def cache_evict(k_pages, v_pages, table, lens, scores, positions, *, budget: int, first: int = 0, recent: int = 0):
    """Bring every sequence down to ``budget`` slots per kv head, by accumulated attention weight.

    Kept are the slots whose position is below ``first`` or among the newest
    ``recent`` positions, and of the others those with the highest ``scores``
    (ties: the lower slot; NaN lowest). ``scores`` float32 and ``positions``
    int32 have shape (B, Hkv, max_pages * page_size). Kept rows at or above the
    budget move, in slot order, into the holes below it; all other rows of the
    cache stay where they are, so the rows moved, not the budget, set the cost.
    A sequence of at most ``budget`` slots is left alone.

    Returns ``(new_lens, new_scores, new_positions, kept)``: new tensors that
    replace ``lens``, ``scores`` and ``positions`` (0 and -1 beyond the new
    length), and ``kept`` (B, Hkv, budget) int32, the old slot of every new one
    (-1: none). The inputs are not changed, so repeating a call repeats its
    result. The pages beyond the new lengths are free afterwards.
    """
    num, Hkv, size, B, maxp, code = _check_cache(k_pages, v_pages, table, lens)
    S = maxp * size
    if not 1 <= budget < 2 ** 31:
        raise ValueError("budget must be positive")
    if first < 0 or recent < 0 or first + recent > budget:
        raise ValueError("first and recent must not be negative and must fit the budget together")
    _check_state("scores", scores, (B, Hkv, S), _F32)
    _check_state("positions", positions, (B, Hkv, S), _I32)
    _same_device(k_pages, v_pages, table, lens, scores, positions)
    dev = k_pages.device
    table, lens = table.contiguous(), lens.contiguous()
    new_lens = torch.empty_like(lens)
    new_scores = torch.empty_like(scores)
    new_positions = torch.empty_like(positions)
    kept = torch.empty((B, Hkv, budget), dtype=_I32, device=dev)
    nbytes = _evict_workspace(B, Hkv, budget)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    L.check(L.lib().algx_cache_evict(
        k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lens.data_ptr(), scores.data_ptr(),
        positions.data_ptr(), budget, first, recent, new_lens.data_ptr(), new_scores.data_ptr(),
        new_positions.data_ptr(), kept.data_ptr(), B, Hkv, num, size, maxp, 64, code, ws.data_ptr(), nbytes,
        L.stream_of(k_pages)), "algx_cache_evict")
    return new_lens, new_scores, new_positions, kept
