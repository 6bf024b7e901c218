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
lengths and positions are read on the device, and one outside its range raises
the device error word (``algx._lib.device_error()``) and is not followed: slots
beyond the table or in a page that does not exist are left out, a length is cut
to the table, a position to the rotary tables' nearest row. No gradients: these are serving operators (the training path
is ``algx.kernels.flash``). The reference has no cache; the formulas are its
QK norm (qk_norm.py:29-43), rotation (algebraic.py:172-179) and attention
weights (algebraic.py:186-216, standard.py:24-38).
"""

from __future__ import annotations

import functools
from typing import Optional

import torch

from .. import _lib as L


def cache_append(qkv, k_pages, v_pages, table, lens, gain_q=None, gain_k=None, *, rotary=None, positions=None,
                 counts=None, slot_positions=None, eps: float = 1e-5):
    """Put the keys and values of T new tokens per sequence into the cache; returns their queries (B, T, Hq, 64).

    ``qkv`` (B, T, Hq + 2 Hkv, 64) holds the [q | k | v] heads of each token
    (the model's packed (B, T, 3, H, 64) projection is its (B, T, 3 H, 64) view).
    ``lens``: slots held before the call; token t goes to slot ``lens[b] + t``
    and the call changes no length. ``gain_q``, ``gain_k`` (64,) float32 apply
    the QK RMS norm, ``rotary`` = (cos, sin), each (rows, 32) float32, the
    rotation at position ``positions[b] + t`` (default: the slot; one outside the
    tables takes their nearest row, and sets the error word). Norm and
    rotation are evaluated in float32 and rounded once. ``counts`` (B,) int32:
    tokens beyond it are padding, stored nowhere, their queries zero.
    ``slot_positions`` (B, Hkv, max_pages * page_size) int32 receives the new
    slots' positions, which ``cache_evict`` reads.
    """
    cos, sin = (None, None) if rotary is None else rotary
    return L.native().cache_append(qkv, k_pages, v_pages, table, lens, gain_q, gain_k, cos, sin, positions, counts,
                                   slot_positions, eps)


@functools.lru_cache(maxsize=256)
def paged_options(kind: str, n: int, c: float, window: Optional[int], first: int):
    """The checked options of one kind of paged attention as the C ABI's configuration holds them:
    kind, n, window, first, scale, inv_unit."""
    if kind not in ("asinh", "softmax"):
        raise ValueError(f"unknown attention kernel: {kind}")
    if kind == "asinh" and (n < 2 or n & (n - 1)):
        raise ValueError("asinh kernel needs n to be a power of two")
    if kind == "asinh" and not (L.has_reciprocal(c) and L.has_reciprocal(8.0 * c)):
        raise ValueError("asinh scale c must be positive and finite")
    if window is not None and not 1 <= window < 2 ** 31:
        raise ValueError("window must be positive")
    if not 0 <= first < 2 ** 31:
        raise ValueError("first must not be negative")
    unit = float(c) if kind == "asinh" else 1.0
    return (L.ALGX_ATTN_ASINH if kind == "asinh" else L.ALGX_ATTN_SOFTMAX, int(n) if kind == "asinh" else 2,
            window or 0, first, 1.0 / (8.0 * unit), 1.0 / unit)


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
    running maximum, so any score whose square float32 holds (below 2^63) is safe.
    A query that sees nothing gives zeros.

    ``scores`` (B, Hkv, max_pages * page_size) float32: the weight every slot
    has received; the call adds its own normalised weights, summed over the
    queries of each kv head, into ``scores_out`` (default: ``scores`` itself) and
    returns ``(o, scores_out)``. The T new slots start from zero, slots beyond
    ``lens`` are set to zero.
    """
    opts = paged_options(kind, n, c, window, first)
    if sink_logit is not None and not isinstance(sink_logit, torch.Tensor):
        sink_logit = torch.as_tensor(sink_logit, dtype=torch.float32)
    if scores is None:
        if scores_out is not None:
            raise ValueError("scores_out without scores")
        return L.native().paged_attention(q, k_pages, v_pages, table, lens, sink_logit, None, None, *opts)
    scores_out = scores if scores_out is None else scores_out
    return L.native().paged_attention(q, k_pages, v_pages, table, lens, sink_logit, scores, scores_out, *opts), scores_out


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
    return L.native().cache_evict(k_pages, v_pages, table, lens, scores, positions, budget, first, recent)
