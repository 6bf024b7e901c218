"""64-bit restatement of the serving operators (paged cache and draft verification).

TEST INFRASTRUCTURE ONLY: the oracle of ``algx.kernels.paged`` and
``algx.kernels.verify``. Plain loops over sequences and heads, written from the
definitions; inputs are CPU tensors whose values are taken as exact.
"""

from __future__ import annotations

import math

import torch

from .reference_math import apply_rotary, int_pow, rho, rms_norm

F64 = torch.float64


def slots_of(pages, table_row, count, head):
    """Rows of the first ``count`` slots of one sequence and head, float64 (count, 64)."""
    size = pages.shape[2]
    rows = [pages[int(table_row[s // size]), head, s % size] for s in range(count)]
    return torch.stack(rows).to(F64) if rows else torch.zeros((0, 64), dtype=F64)


def sees(slot: int, last: int, window, first: int) -> bool:
    """Whether a query standing at slot ``last`` sees ``slot``."""
    return slot <= last and (not window or slot > last - window or slot < first)


def weights(x, sink, kind: str, n: int):
    """Normalised weights of the visible scores ``x`` (1-d, float64); ``sink`` None or a score in the same unit."""
    every = x if sink is None else torch.cat([x, torch.as_tensor([sink], dtype=F64)])
    if every.numel() == 0:
        return x
    m = every.max()
    w = int_pow(rho(every) * rho(-m), n) if kind == "asinh" else torch.exp(every - m)
    return w[:x.numel()] / w.sum()


def paged_attention(q, k_pages, v_pages, table, lens, sink=None, *, kind="asinh", n=16, c=16.0, window=None, first=0,
                    scores=None):
    """(o, new scores or None, sum of weight |v| per output, largest |score|)."""
    B, T, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    G = Hq // Hkv
    unit = c if kind == "asinh" else 1.0
    o = torch.zeros((B, T, Hq, D), dtype=F64)
    mag = torch.zeros_like(o)
    S = table.shape[1] * k_pages.shape[2]
    out = torch.zeros((B, Hkv, S), dtype=F64)
    top = 0.0
    for b in range(B):
        length = max(0, int(lens[b]))
        for h in range(Hkv):
            k, v = (slots_of(p, table[b], length, h) for p in (k_pages, v_pages))
            if scores is not None:
                old = max(0, length - T)
                out[b, h, :old] = scores[b, h, :old].to(F64)
            for t in range(T):
                seen = [s for s in range(length) if sees(s, length - T + t, window, first)]
                for g in range(G):
                    j = h * G + g
                    x = (k[seen] @ q[b, t, j].to(F64)) / (math.sqrt(D) * unit)
                    p = weights(x, None if sink is None else float(sink[j]) / unit, kind, n)
                    o[b, t, j] = p @ v[seen]
                    mag[b, t, j] = p @ v[seen].abs()
                    if seen:
                        out[b, h, seen] += p
                        top = max(top, float(x.abs().max()))
    return o, (None if scores is None else out), mag, top


def cache_append(qkv, k_pages, v_pages, table, lens, gain_q=None, gain_k=None, *, rotary=None, positions=None,
                 counts=None, eps=1e-5):
    """(q, k_pages, v_pages) in float64; the given pages are copied, not changed."""
    B, T, _, D = qkv.shape
    Hkv, size = k_pages.shape[1], k_pages.shape[2]
    Hq = qkv.shape[2] - 2 * Hkv
    kp, vp = k_pages.to(F64).clone(), v_pages.to(F64).clone()
    q = torch.zeros((B, T, Hq, D), dtype=F64)

    def turn(x, gain, pos):
        y = x.to(F64) if gain is None else rms_norm(x.to(F64), gain.to(F64), eps)
        if rotary is None:
            return y
        cos, sin = (r[pos:pos + 1].to(F64) for r in rotary)
        return apply_rotary(y[None, :, None], cos, sin)[0, :, 0]

    for b in range(B):
        for t in range(T if counts is None else min(T, int(counts[b]))):
            slot = int(lens[b]) + t
            pos = (int(lens[b]) if positions is None else int(positions[b])) + t
            x = qkv[b, t]
            q[b, t] = turn(x[:Hq], gain_q, pos)
            page = int(table[b, slot // size])
            kp[page, :, slot % size] = turn(x[Hq:Hq + Hkv], gain_k, pos)
            vp[page, :, slot % size] = x[Hq + Hkv:].to(F64)
    return q, kp, vp


def evict_plan(scores, positions, length: int, budget: int, first: int, recent: int):
    """Old slot of every new slot for one sequence and head (1-d scores and positions)."""
    if length <= budget:
        return list(range(length))
    newest = max(int(p) for p in positions[:length])

    def rank(s):  # protected slots, then scores from the highest on, then NaN
        p, x = int(positions[s]), float(scores[s])
        if p < first or p > newest - recent:
            return (0, 0.0, s)
        return (2, 0.0, s) if math.isnan(x) else (1, -x, s)

    keep = sorted(sorted(range(length), key=rank)[:budget])
    held = set(keep)
    movers = iter(s for s in keep if s >= budget)
    return [s if s in held else next(movers) for s in range(budget)]


def probabilities(z, kind: str, n: int, c: float, temperature: float = 1.0):
    """Row probabilities of 1-d logits, zero at -inf and NaN; all zero where nothing is left.

    The operator's probabilities are float32 numbers, of which the smallest is
    2^-149: one below 2^-150 is zero."""
    z = z.to(F64)
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    if not bool((z > -math.inf).any()):
        return torch.zeros_like(z)
    if kind == "ce":
        p = torch.softmax(z / temperature, dim=-1)
        return torch.where(p < 2.0 ** -150, torch.zeros_like(p), p)
    x = torch.where(z > -math.inf, z, torch.zeros_like(z)) / c
    m = x[z > -math.inf].max()
    w = torch.where(z > -math.inf, int_pow(rho(x) * rho(-m), n), torch.zeros_like(x))
    p = w / w.sum()
    return torch.where(p < 2.0 ** -150, torch.zeros_like(p), p)


def verify_draft(target, tokens, draft, u, race, *, kind="ce", n=16, c=16.0, temperature=1.0, counts=None):
    """(tokens, accepted) as nested lists."""
    B, rows, V = target.shape
    out, accepted = [], []
    for b in range(B):
        K = rows - 1 if counts is None else max(0, min(int(counts[b]), rows - 1))
        taken, left = [], None
        for i in range(K):
            p = probabilities(target[b, i], kind, n, c, temperature)
            x = int(tokens[b, i])
            ok = 0 <= x < V
            if draft is not None:
                q = probabilities(draft[b, i], kind, n, c, temperature)
            else:
                q = torch.zeros(V, dtype=F64)
                if ok:
                    q[x] = 1.0
            if ok and float(u[b, i]) * float(q[x]) < float(p[x]):
                taken.append(x)
                continue
            left = torch.clamp(p - q, min=0)
            if not bool((left > 0).any()):
                left = p
            break
        if left is None:
            left = probabilities(target[b, K], kind, n, c, temperature)
        ratio = torch.where(left > 0, left / race[b].to(F64), torch.zeros_like(left))
        accepted.append(len(taken))
        out.append(taken + [int(torch.argmax(ratio))] + [-1] * (rows - 1 - len(taken)))
    return out, accepted
