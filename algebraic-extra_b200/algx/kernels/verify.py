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

import functools

from .. import _lib as L


@functools.lru_cache(maxsize=256)
def _options(kind: str, n: int, c: float, temperature: float):
    """The checked options as the C ABI takes them: kind, n, scale."""
    if kind not in ("ce", "alg_ce"):
        raise ValueError(kind)
    if kind == "alg_ce":
        if n not in (2, 4, 8, 16, 32):
            raise ValueError("algx supports alg_ce powers n in {2, 4, 8, 16, 32}")
        if not L.has_reciprocal(c):
            raise ValueError("alg_ce scale c must be positive and finite")
        if temperature != 1.0:
            raise ValueError("temperature is for the ce kind")
        return L.ALGX_HEAD_ALG_CE, n, 1.0 / c
    if not L.has_reciprocal(temperature):
        raise ValueError("temperature must be positive and finite")
    return L.ALGX_HEAD_CE, 2, 1.0 / temperature


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
    have probability 0, and so have NaN ones; alg_ce takes ``|z / c|`` below 2^63,
    whose square float32 holds. ``temperature`` divides the logits of the ``ce`` kind. ``counts`` (B,) int32: drafts of each
    sequence where not all have K (row ``counts[b]`` is then the one after).

    ``tokens`` (B, K + 1) int32 holds the accepted drafts, the token drawn, then
    -1; ``accepted`` (B,) int32. A draft token outside [0, V) is refused and
    raises the device error word (``algx._lib.device_error()``).
    """
    return L.native().verify_draft(target_logits, draft_tokens, draft_logits, accept_u, race, counts,
                                   *_options(kind, n, c, temperature))
