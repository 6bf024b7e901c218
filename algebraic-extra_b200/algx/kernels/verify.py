"""Verification of drafted tokens and the draw of the next one, under either likelihood head.

``verify_draft`` takes the target model's logits for K drafted tokens and the
token after them, the draft model's logits, and the random numbers, and returns
how many drafts are accepted and which token follows. The output tokens are
distributed as the target model's own samples. With K = 0 it samples one token.
Probabilities are those of the framework's heads: softmax (``ce``) or
rho(z / c)^n normalised (``alg_ce``, algebraic.py:266-301). The reference has no
counterpart.
"""

from __future__ import annotations

import math

import torch

from .. import _lib as L

_CODE = {torch.bfloat16: L.ALGX_BF16, torch.float32: L.ALGX_F32}


def verify_draft(target_logits, draft_tokens, draft_logits, accept_u, race, *, kind: str = "ce", n: int = 16,
                 c: float = 16.0, temperature: float = 1.0, counts=None):
    """Accept drafted tokens against the target's probabilities; returns (tokens, accepted).

    ``target_logits`` (B, K + 1, V) and ``draft_logits`` (B, K, V), bfloat16 or
    float32; ``draft_logits`` None means certain proposals (a lookup, not a
    model: q = 1 at the drafted token). ``draft_tokens`` (B, K) int32, drawn from
    the draft's probabilities, ``accept_u`` (B, K) float32 uniform on [0, 1), ``race`` (B, V) float32
    exponential variates. K is at most 31.

    Draft i is accepted while ``accept_u[b, i] * q_i(x_i) < p_i(x_i)``. After the
    first refusal the next token is drawn from max(p - q, 0) of that row, after
    K acceptances from row K, as the argmax of weight / race (ties: the lowest
    index). Probabilities are float32 numbers (below 2^-150: zero); -inf logits
    have probability 0, and so have NaN ones. ``temperature``
    divides the logits of the ``ce`` kind. ``counts`` (B,) int32: drafts of each
    sequence where not all have K (row ``counts[b]`` is then the one after).

    ``tokens`` (B, K + 1) int32 holds the accepted drafts, the token drawn, then
    -1; ``accepted`` (B,) int32. A draft token outside [0, V) is refused and
    raises the device error word (``algx._lib.device_error()``).
    """
    if kind not in ("ce", "alg_ce"):
        raise ValueError(kind)
    if kind == "alg_ce":
        if n not in (2, 4, 8, 16, 32):
            raise ValueError("algx supports alg_ce powers n in {2, 4, 8, 16, 32}")
        if not math.isfinite(c) or c <= 0:
            raise ValueError("alg_ce scale c must be positive and finite")
        if temperature != 1.0:
            raise ValueError("temperature is for the ce kind")
    if not math.isfinite(temperature) or temperature <= 0:
        raise ValueError("temperature must be positive and finite")
    shape, dtype = target_logits.shape, target_logits.dtype
    if len(shape) != 3 or shape[1] < 1 or shape[2] < 1:
        raise ValueError(f"target_logits must have shape (B, K + 1, V), got {tuple(shape)}")
    B, K, V = shape[0], shape[1] - 1, shape[2]
    if K > 31:
        raise ValueError("at most 31 drafted tokens")
    io = _CODE.get(dtype)
    if io is None:
        raise ValueError("logits must be bfloat16 or float32")
    if draft_logits is not None and (draft_logits.shape != (B, K, V) or draft_logits.dtype != dtype):
        raise ValueError(f"draft_logits must have shape {(B, K, V)} and target_logits' dtype")
    if draft_tokens.shape != (B, K) or draft_tokens.dtype != torch.int32:
        raise ValueError(f"draft_tokens must be int32 of shape {(B, K)}")
    if accept_u.shape != (B, K) or accept_u.dtype != torch.float32:
        raise ValueError(f"accept_u must be float32 of shape {(B, K)}")
    if race.shape != (B, V) or race.dtype != torch.float32:
        raise ValueError(f"race must be float32 of shape {(B, V)}")
    if counts is not None and (counts.shape != (B,) or counts.dtype != torch.int32):
        raise ValueError(f"counts must be int32 of shape ({B},)")
    dev = target_logits.get_device()
    for t in (draft_logits, draft_tokens, accept_u, race, counts):
        if t is not None and t.get_device() != dev:
            L.require_cuda(target_logits, t)
            raise ValueError(f"tensors on {target_logits.device} and {t.device} in one call")
    L.require_cuda(target_logits)
    target, draft_tokens, accept_u, race = (t.contiguous() for t in (target_logits, draft_tokens, accept_u, race))
    draft = None if draft_logits is None else draft_logits.contiguous()
    counts = None if counts is None else counts.contiguous()
    device = target.device
    tokens = torch.empty((B, K + 1), dtype=torch.int32, device=device)
    accepted = torch.empty(B, dtype=torch.int32, device=device)
    code, scale = (L.ALGX_HEAD_CE, 1.0 / temperature) if kind == "ce" else (L.ALGX_HEAD_ALG_CE, 1.0 / c)
    L.check(L.lib().algx_verify_draft(
        code, n, scale, target.data_ptr(), L.ptr(draft), draft_tokens.data_ptr(), L.ptr(counts), accept_u.data_ptr(),
        race.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), B, K, V, io, L.stream_of(target)), "algx_verify_draft")
    return tokens, accepted
