"""Timed cases of the serving operators: cache append, paged attention, cache eviction and draft verification.

``listed()`` names the cases, ``draw(rng)`` makes another one of the same ranges, ``prepare`` builds what a serving
loop has in hand before the call, and ``run`` makes one call: in plain torch operations when ``own`` is False, through
``algx.kernels.paged`` and ``algx.kernels.verify`` when it is True. ``exact`` restates the definitions in 64 bits.

Shapes follow the framework's models: head width 64, 12 heads (125M) or 16 (350M), a vocabulary of 50304, sequences of
2048 tokens, attention n = 16, c = 8; grouped heads, longer caches and other vocabularies stand for what a serving
loop meets beyond them.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

D = 64
EPS = 1e-5
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}


def _algx():
    root = os.path.join(os.getcwd(), "algebraic-extra_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from algx.kernels import paged, verify
    return paged, verify


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of one sequence enters the cache: the smallest call of a decode step
        _append("append one token", B=1, T=1, Hq=12, Hkv=12, cap=2048, page=64, dtype="bf16"),
        # eight prompts of 2048 tokens enter the cache after prefill
        _append("append prompts", B=8, T=2048, Hq=12, Hkv=12, cap=2304, page=64, dtype="bf16"),
        # one user, the 125M model at its training length: latency
        _attend("attend one user", B=1, T=1, Hq=12, Hkv=12, cap=2048, page=64, dtype="bf16", kind="asinh", n=16, c=8.0),
        # a batch of ragged sequences with the learned sink, accumulating the weights that eviction reads
        _attend("attend batch scored", B=32, T=1, Hq=12, Hkv=12, cap=2048, page=64, dtype="bf16", kind="asinh", n=16,
                c=8.0, sink=True, scored=True, ragged=5),
        # five tokens per sequence (four drafted) against grouped heads: the target's pass of speculative decoding
        _attend("attend drafts grouped", B=16, T=5, Hq=32, Hkv=8, cap=8192, page=64, dtype="bf16", kind="softmax",
                n=16, c=16.0, ragged=11),
        # long documents: the largest case, read once from end to end
        _attend("attend long", B=8, T=1, Hq=16, Hkv=16, cap=32768, page=128, dtype="bf16", kind="asinh", n=16, c=8.0,
                ragged=3),
        # sliding window with four first tokens left visible in a long cache
        _attend("attend window", B=32, T=1, Hq=16, Hkv=16, cap=16384, page=16, dtype="bf16", kind="asinh", n=16, c=8.0,
                sink=True, window=1024, first=4, ragged=7),
        # float32 cache, odd length: evaluation runs
        _attend("attend float32", B=4, T=1, Hq=12, Hkv=12, cap=4096, page=32, dtype="f32", kind="asinh", n=16, c=8.0,
                ragged=13),
        # one sequence over its budget
        _evict("evict one user", B=1, Hkv=12, cap=2560, page=64, budget=2048, first=4, recent=256, dtype="bf16",
               full=True),
        # a batch brought down to half its length
        _evict("evict batch", B=16, Hkv=12, cap=8192, page=64, budget=4096, first=4, recent=512, dtype="bf16",
               full=True),
        # four drafted tokens of one user
        _verify("verify one user", B=1, K=4, V=50304, dtype="bf16", kind="ce", n=16, c=16.0),
        # a batch with seven drafted tokens each under the algebraic likelihood head
        _verify("verify batch", B=64, K=7, V=50304, dtype="f32", kind="alg_ce", n=8, c=2.0),
    ]


def _append(name, B, T, Hq, Hkv, cap, page, dtype):
    return {"name": name, "op": "append", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "cap": cap, "page": page,
            "dtype": dtype}


def _attend(name, B, T, Hq, Hkv, cap, page, dtype, kind, n, c, sink=False, scored=False, window=0, first=0, ragged=0):
    return {"name": name, "op": "attend", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "cap": cap, "page": page,
            "dtype": dtype, "kind": kind, "n": n, "c": c, "sink": sink, "scored": scored, "window": window,
            "first": first, "ragged": ragged}


def _evict(name, B, Hkv, cap, page, budget, first, recent, dtype, full):
    return {"name": name, "op": "evict", "B": B, "Hkv": Hkv, "cap": cap, "page": page, "budget": budget,
            "first": first, "recent": recent, "dtype": dtype, "full": full}


def _verify(name, B, K, V, dtype, kind, n, c):
    return {"name": name, "op": "verify", "B": B, "K": K, "V": V, "dtype": dtype, "kind": kind, "n": n, "c": c}


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "verify"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    page = rng.choice([16, 32, 64, 128, 256])
    Hkv = rng.choice([1, 2, 3, 4, 8, 12, 16])
    G = rng.choice([1, 1, 1, 2, 4, 5, 8])
    if op == "append":
        B = _logint(rng, 1, 64)
        T = _logint(rng, 1, max(1, 16384 * 36 // (B * Hkv * (G + 2))) if B * Hkv * (G + 2) < 16384 else 1)
        T = min(T, 2048)
        case = _append("", B, T, Hkv * G, Hkv, T + _logint(rng, 1, 512), page, dtype)
    elif op == "attend":
        B = _logint(rng, 1, 64)
        T = rng.choice([1, 1, 1, 2, 3, 5, 9])
        # at most the slots x heads (bytes) and score products of the largest listed case
        most = 8 * 32768 * 16 * 2 // (B * Hkv * SIZE[dtype] * max(1, G * T // 8))
        cap = max(T, _logint(rng, 16, min(65536, max(17, most))))
        kind = rng.choice(["asinh", "asinh", "softmax"])
        window = rng.choice([0, 0, _logint(rng, 1, 2048)])
        case = _attend("", B, T, Hkv * G, Hkv, cap, page, dtype, kind, rng.choice([2, 4, 8, 16, 32]),
                       rng.choice([2.0, 8.0, 16.0]), sink=rng.random() < 0.5,
                       scored=rng.random() < 0.3, window=window, first=rng.choice([0, 1, 4, 9]) if window else 0,
                       ragged=rng.randrange(1, 1000))
    elif op == "evict":
        B = _logint(rng, 1, 32)
        cap = _logint(rng, 64, max(65, min(32768, 16 * 12 * 8192 // (B * Hkv))))
        budget = rng.randrange(32, cap + 1)
        first = rng.choice([0, 1, 4])
        case = _evict("", B, Hkv, cap, page, budget, first, rng.randrange(0, max(1, (budget - first) // 2)), dtype,
                      rng.random() < 0.5)
    else:
        B = _logint(rng, 1, 64)
        V = rng.choice([50304, 32000, _logint(rng, 257, 50304)])
        case = _verify("", B, rng.randrange(1, 8), V, dtype, rng.choice(["ce", "alg_ce"]), rng.choice([2, 4, 8, 16, 32]),
                       rng.choice([2.0, 4.0, 16.0]))
    del case["name"]
    return case


def _lens(case):
    """Cached slots per sequence: all full, or spread over the range by a fixed rule."""
    B, cap = case["B"], case["cap"]
    if case["op"] == "append":
        return [(cap - case["T"]) * (b + 1) // B for b in range(B)]
    if case["op"] == "evict":
        return [cap if case["full"] else 1 + (cap - 1) * ((7 * b + 3) % B + 1) // B for b in range(B)]
    if not case["ragged"]:
        return [cap] * B
    lo = case["T"] if cap > case["T"] else cap
    return [cap if b == 0 else lo + (case["ragged"] * 7919 * b + 104729 * b * b) % (cap - lo + 1) for b in range(B)]


# ------------------------------------------------------------------ inputs
def _pages_of(case):
    return -(-case["cap"] // case["page"])


def _cache(case, gen, fill):
    """Paged cache whose pages lie in no order, as after some time of serving; about a tenth of the pages are free."""
    B, P, Hkv, page = case["B"], _pages_of(case), case["Hkv"], case["page"]
    num = B * P + max(1, B * P // 10)
    shape = (num, Hkv, page, D)
    if fill:
        k = torch.randn(shape, generator=gen, device="cuda", dtype=DT[case["dtype"]])
        v = torch.randn(shape, generator=gen, device="cuda", dtype=DT[case["dtype"]])
    else:
        k = torch.zeros(shape, device="cuda", dtype=DT[case["dtype"]])
        v = torch.zeros(shape, device="cuda", dtype=DT[case["dtype"]])
    table = torch.randperm(num, generator=gen, device="cuda")[:B * P].reshape(B, P).to(torch.int32).contiguous()
    return k, v, table


def _rope(rows):
    theta = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * theta
    return torch.cos(ang).float().cuda(), torch.sin(ang).float().cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT.get(case["dtype"])
    st = {"case": dict(case)}
    if case["op"] == "verify":
        B, K, V = case["B"], case["K"], case["V"]
        # logits with a few likely tokens, and a draft model that agrees with the target in part
        base = torch.randn((B, K + 1, V), generator=gen, device="cuda") * 2.0
        base[:, :, :16] += 6.0
        scale = 1.0 if case["kind"] == "ce" else case["c"]
        st["target"] = (base * scale).to(dt)
        noise = torch.randn((B, K, V), generator=gen, device="cuda") * 0.7
        draft = (base[:, :K] + noise) * scale
        st["draft"] = draft.to(dt)
        prob = torch.softmax(draft / scale, dim=-1).reshape(B * K, V)
        st["tokens"] = torch.multinomial(prob, 1, generator=gen).reshape(B, K).to(torch.int32)
        st["u"] = torch.rand((B, K), generator=gen, device="cuda")
        st["race"] = -torch.log1p(-torch.rand((B, V), generator=gen, device="cuda").clamp_(1e-7, 1 - 1e-7))
        return st
    st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    st["k"], st["v"], st["table"] = _cache(case, gen, fill=case["op"] != "append")
    if case["op"] == "append":
        B, T, H = case["B"], case["T"], case["Hq"] + 2 * case["Hkv"]
        st["qkv"] = torch.randn((B, T, H, D), generator=gen, device="cuda").to(dt)
        st["gain_q"] = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
        st["gain_k"] = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
        st["rot"] = _rope(case["cap"])
        return st
    S = _pages_of(case) * case["page"]
    if case["op"] == "attend":
        st["q"] = torch.randn((case["B"], case["T"], case["Hq"], D), generator=gen, device="cuda").to(dt)
        st["sink"] = torch.randn(case["Hq"], generator=gen, device="cuda") * case["c"] if case["sink"] else None
        if case["scored"]:
            st["scores"] = torch.rand((case["B"], case["Hkv"], S), generator=gen, device="cuda")
            st["scores_out"] = torch.empty_like(st["scores"])
        return st
    # eviction: a few slots hold most of the weight, and slots are not in the order of their positions
    shape = (case["B"], case["Hkv"], S)
    st["scores"] = torch.rand(shape, generator=gen, device="cuda") ** 8
    noise = torch.rand(shape, generator=gen, device="cuda")
    noise = torch.where(torch.arange(S, device="cuda") < st["lens"][:, None, None], noise, 2.0)
    st["positions"] = torch.argsort(torch.argsort(noise, dim=-1), dim=-1).to(torch.int32)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    op = st["case"]["op"]
    if own:
        paged, verify = _algx()
        if op == "append":
            q = paged.cache_append(st["qkv"], st["k"], st["v"], st["table"], st["lens"], st["gain_q"], st["gain_k"],
                                   rotary=st["rot"], eps=EPS)
            return q, st["k"], st["v"]
        if op == "attend":
            c = st["case"]
            kw = dict(kind=c["kind"], n=c["n"], c=c["c"], window=c["window"] or None, first=c["first"])
            if c["scored"]:
                return paged.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], st["sink"],
                                             scores=st["scores"], scores_out=st["scores_out"], **kw)
            return paged.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], st["sink"], **kw)
        if op == "evict":
            c = st["case"]
            out = paged.cache_evict(st["k"], st["v"], st["table"], st["lens"], st["scores"], st["positions"],
                                    budget=c["budget"], first=c["first"], recent=c["recent"])
            return (*out, st["k"], st["v"])
        c = st["case"]
        return verify.verify_draft(st["target"], st["tokens"], st["draft"], st["u"], st["race"], kind=c["kind"],
                                   n=c["n"], c=c["c"])
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "verify": _plain_verify}[op](st)


def _where(st, slots):
    """(page, offset) of slots (B, ...) through the page table."""
    page = st["case"]["page"]
    flat = slots.reshape(slots.shape[0], -1)
    pages = torch.gather(st["table"].long(), 1, torch.div(flat, page, rounding_mode="floor"))
    return pages.reshape(slots.shape), slots % page


def _plain_append(st):
    c = st["case"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    x = st["qkv"].float()
    pos = st["lens"].long()[:, None] + torch.arange(c["T"], device=x.device)
    cos, sin = (t[pos][:, :, None] for t in st["rot"])

    def turn(y, gain):
        y = y * torch.rsqrt(torch.mean(y * y, dim=-1, keepdim=True) + EPS) * gain
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1).to(st["qkv"].dtype)

    page, off = _where(st, pos)
    st["k"][page, :, off] = turn(x[:, :, Hq:Hq + Hkv], st["gain_k"])
    st["v"][page, :, off] = st["qkv"][:, :, Hq + Hkv:]
    return turn(x[:, :, :Hq], st["gain_q"]), st["k"], st["v"]


def _power(x, n):
    return x if n == 1 else _power(x * x, n // 2)


def _rho(x):
    t = torch.abs(x) + torch.sqrt(1 + x * x)
    return torch.where(x >= 0, t, 1 / t)


def _plain_attend(st):
    c = st["case"]
    B, T, Hq, Hkv = c["B"], c["T"], c["Hq"], c["Hkv"]
    G = Hq // Hkv
    table = st["table"].long()
    k = st["k"][table].transpose(1, 2).reshape(B, Hkv, -1, D).float()
    v = st["v"][table].transpose(1, 2).reshape(B, Hkv, -1, D).float()
    S = k.shape[2]
    q = st["q"].float().reshape(B, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, D)
    unit = c["c"] if c["kind"] == "asinh" else 1.0
    x = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / (math.sqrt(D) * unit))
    slot = torch.arange(S, device=x.device)
    last = (st["lens"].long()[:, None] - T + torch.arange(T, device=x.device)).repeat_interleave(G, dim=1)
    last = last[:, None, :, None]
    see = slot <= last
    if c["window"]:
        see = see & ((slot > last - c["window"]) | (slot < c["first"]))
    m = torch.where(see, x, -math.inf).amax(dim=-1, keepdim=True)
    if st["sink"] is not None:
        b = (st["sink"] / unit).reshape(1, Hkv, 1, G).expand(B, Hkv, T, G).reshape(B, Hkv, T * G, 1)
        m = torch.maximum(m, b)
    m = torch.where(torch.isfinite(m), m, 0.0)
    if c["kind"] == "asinh":
        turn = _rho(-m)
        weight = lambda y: _power(_rho(y) * turn, c["n"])  # noqa: E731
    else:
        weight = lambda y: torch.exp(y - m)  # noqa: E731
    w = torch.where(see, weight(x), 0.0)
    total = w.sum(dim=-1, keepdim=True)
    if st["sink"] is not None:
        total = total + weight(b)
    p = w / torch.where(total > 0, total, 1.0)
    v = torch.where((slot < st["lens"][:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(p, v).reshape(B, Hkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, Hq, D).to(st["q"].dtype)
    if not c["scored"]:
        return o
    old = torch.where(slot < (st["lens"][:, None, None] - T), st["scores"], 0.0)
    st["scores_out"].copy_(old + p.sum(dim=2))
    return o, st["scores_out"]


def _plain_evict(st):
    c = st["case"]
    budget = c["budget"]
    scores, positions, lens = st["scores"], st["positions"], st["lens"]
    S = scores.shape[-1]
    slot = torch.arange(S, device=scores.device)
    live = slot < lens[:, None, None]
    newest = torch.where(live, positions, -1).amax(dim=-1, keepdim=True)
    kept_always = (positions < c["first"]) | (positions > newest - c["recent"])
    key = torch.where(live, torch.where(kept_always, math.inf, scores), -math.inf)
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order).contiguous())
    keep = live & (rank < budget)
    # the i-th kept slot at or above the budget goes to the i-th hole below it
    hole = ~keep & (slot < budget) & (slot < lens[:, None, None])
    mover = keep & (slot >= budget)
    movers = torch.where(mover, slot, S).sort(dim=-1).values
    nth = torch.cumsum(hole, dim=-1) - 1
    source = torch.where(hole, torch.gather(movers, -1, nth.clamp(min=0)), slot)
    new_lens = torch.minimum(lens, torch.full_like(lens, budget))
    stays = slot < new_lens[:, None, None]
    source = torch.where(stays, source, 0)
    new_scores = torch.where(stays, torch.gather(scores, -1, source), 0.0)
    new_positions = torch.where(stays, torch.gather(positions, -1, source), -1)
    B, H = scores.shape[:2]
    sp, so = _where(st, source)
    dp, do = _where(st, slot.expand(B, H, S))
    head = torch.arange(H, device=scores.device)[None, :, None].expand(B, H, S)
    b, h, s = torch.nonzero(hole, as_tuple=True)
    at = (dp[b, h, s], head[b, h, s], do[b, h, s])
    of = (sp[b, h, s], head[b, h, s], so[b, h, s])
    st["k"][at] = st["k"][of]
    st["v"][at] = st["v"][of]
    kept = torch.where(stays, source, -1)[..., :budget].to(torch.int32).contiguous()
    return new_lens, new_scores, new_positions.to(torch.int32), kept, st["k"], st["v"]


def _plain_probs(z, kind, n, c):
    z = z.float()
    if kind == "ce":
        w = torch.exp(z - z.amax(dim=-1, keepdim=True))
    else:
        x = z * (1.0 / c)
        w = _power(_rho(x) * _rho(-x.amax(dim=-1, keepdim=True)), n)
    return w / w.sum(dim=-1, keepdim=True)


def _plain_verify(st):
    c = st["case"]
    B, K = c["B"], c["K"]
    p = _plain_probs(st["target"], c["kind"], c["n"], c["c"])
    q = _plain_probs(st["draft"], c["kind"], c["n"], c["c"])
    tok = st["tokens"].long()[:, :, None]
    ok = st["u"] * torch.gather(q, 2, tok)[..., 0] < torch.gather(p[:, :K], 2, tok)[..., 0]
    accepted = torch.cumprod(ok.int(), dim=1).sum(dim=1)
    row = torch.arange(B, device=p.device)
    base = p[row, accepted]
    rest = torch.clamp(base - q[row, accepted.clamp(max=K - 1)], min=0.0)
    use = (accepted < K) & (rest.amax(dim=-1) > 0)
    pick = torch.argmax(torch.where(use[:, None], rest, base) / st["race"], dim=-1)
    at = torch.arange(K + 1, device=p.device)
    drafted = torch.cat([st["tokens"], torch.zeros_like(st["tokens"][:, :1])], dim=1)
    tokens = torch.where(at < accepted[:, None], drafted, torch.where(at == accepted[:, None], pick[:, None], -1))
    return tokens.to(torch.int32), accepted.to(torch.int32)


# ------------------------------------------------------------------ the least work
def work(case):
    B, e = case["B"], SIZE[case["dtype"]]
    if case["op"] == "append":
        rows = B * case["T"] * (case["Hq"] + 2 * case["Hkv"])
        return {"bytes": 2 * rows * D * e + B * case["T"] * D * 4, "flops": 8 * rows * D}
    if case["op"] == "verify":
        K, V = case["K"], case["V"]
        rows = B * (2 * K + 1)
        return {"bytes": rows * V * e + B * V * 4, "flops": 8 * rows * V}
    Hkv, lens = case["Hkv"], _lens(case)
    if case["op"] == "attend":
        T, Hq = case["T"], case["Hq"]
        slots = [n if not case["window"] else min(n, case["window"] + T - 1 + min(case["first"], n)) for n in lens]
        total = sum(slots)
        S = _pages_of(case) * case["page"]
        nbytes = 2 * total * Hkv * D * e + 2 * B * T * Hq * D * e
        if case["scored"]:
            nbytes += Hkv * 4 * (sum(lens) + B * S)
        return {"bytes": nbytes, "flops": 4 * D * T * Hq * total}
    budget, first, recent = case["budget"], case["first"], case["recent"]
    S = _pages_of(case) * case["page"]
    moved = 0.0
    for n in lens:
        if n > budget:
            held = min(budget, first + recent)
            moved += (n - budget) * (held / n + (1 - held / n) * (budget - held) / max(1, n - held))
    nbytes = Hkv * (8 * sum(lens) + B * (8 * S + 4 * budget)) + int(moved * Hkv) * 4 * D * e
    return {"bytes": nbytes, "flops": 4 * Hkv * sum(lens)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict, "verify": _exact_verify}[
        case["op"]](case, st)


def _exact_append(case, st):
    Hq, Hkv, page = case["Hq"], case["Hkv"], case["page"]
    k, v = st["k"].double(), st["v"].double()
    rows = []
    for b, start in enumerate(_lens(case)):
        x = st["qkv"][b].double()
        at = torch.arange(start, start + case["T"], device=x.device)
        turn = torch.complex(st["rot"][0][at].double(), st["rot"][1][at].double())[:, None]

        def rotated(y, gain):
            y = y / torch.linalg.vector_norm(y, dim=-1, keepdim=True).square().div(D).add(EPS).sqrt() * gain.double()
            z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], dim=-1)

        pages, off = st["table"][b].long()[at // page], at % page
        k[pages, :, off] = rotated(x[:, Hq:Hq + Hkv], st["gain_k"])
        v[pages, :, off] = x[:, Hq + Hkv:]
        rows.append(rotated(x[:, :Hq], st["gain_q"]))
    return torch.stack(rows), k, v


def _exact_attend(case, st):
    T, Hq, Hkv, n = case["T"], case["Hq"], case["Hkv"], case["n"]
    G = Hq // Hkv
    unit = case["c"] if case["kind"] == "asinh" else 1.0
    outs, news = [], []
    for b, length in enumerate(_lens(case)):
        pages = st["table"][b].long()
        k = st["k"][pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :length].double()
        v = st["v"][pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :length].double()
        q = st["q"][b].double().reshape(T, Hkv, G, D)
        x = torch.einsum("thgd,hsd->htgs", q, k) / (math.sqrt(D) * unit)
        s = torch.arange(length, device=x.device)[None, :]
        t = torch.arange(length - T, length, device=x.device)[:, None]
        hidden = s > t
        if case["window"]:
            hidden = hidden | ((t - s >= case["window"]) & (s >= case["first"]))
        # log-weights: n asinh(x) or x; the sink is one more column
        logw = n * torch.asinh(x) if case["kind"] == "asinh" else x
        logw = logw.masked_fill(hidden[None, :, None, :], -math.inf)
        if st["sink"] is not None:
            y = (st["sink"].double() / unit).reshape(Hkv, 1, G, 1).expand(Hkv, T, G, 1)
            logw = torch.cat([logw, n * torch.asinh(y) if case["kind"] == "asinh" else y], dim=-1)
        p = torch.softmax(logw, dim=-1)[..., :length]
        p = torch.nan_to_num(p, nan=0.0)
        outs.append(torch.einsum("htgs,hsd->thgd", p, v).reshape(T, Hq, D))
        if case["scored"]:
            old = st["scores"][b].double().clone()
            old[:, max(0, length - T):] = 0
            old[:, :length] += p.sum(dim=(1, 2))
            news.append(old)
    o = torch.stack(outs)
    return (o, torch.stack(news)) if case["scored"] else o


def _exact_evict(case, st):
    budget, first, recent, page = case["budget"], case["first"], case["recent"], case["page"]
    lens = _lens(case)
    scores, positions = st["scores"].double().cpu().numpy(), st["positions"].cpu().numpy()
    table = st["table"].cpu().numpy()
    new_scores, new_positions = np.zeros_like(scores), np.full_like(positions, -1)
    kept = np.full(scores.shape[:2] + (budget,), -1, dtype=np.int32)
    moves = []
    for b, n in enumerate(lens):
        for h in range(case["Hkv"]):
            sc, po = scores[b, h, :n].copy(), positions[b, h, :n]
            if n <= budget:
                src = np.arange(n)
            else:
                sc[(po < first) | (po > po.max() - recent)] = np.inf
                chosen = np.sort(np.lexsort((np.arange(n), -sc))[:budget])
                src = np.arange(budget)
                gone = np.setdiff1d(src, chosen)
                src[gone] = chosen[chosen >= budget]
                for to in gone:
                    moves.append((table[b, to // page], h, to % page, table[b, src[to] // page], src[to] % page))
            kept[b, h, :len(src)] = src
            new_scores[b, h, :len(src)] = scores[b, h, src]
            new_positions[b, h, :len(src)] = positions[b, h, src]
    k, v = st["k"].double(), st["v"].double()
    if moves:
        tp, h, to, fp, fo = torch.as_tensor(np.array(moves, dtype=np.int64), device=k.device).unbind(1)
        k[tp, h, to] = k[fp, h, fo]
        v[tp, h, to] = v[fp, h, fo]
    as_t = lambda a: torch.as_tensor(a, device=k.device)  # noqa: E731
    new_lens = torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=k.device)
    return new_lens, as_t(new_scores), as_t(new_positions), as_t(kept), k, v


def _exact_verify(case, st):
    def probs(z):
        z = z.double()
        return torch.softmax(z if case["kind"] == "ce" else case["n"] * torch.asinh(z / case["c"]), dim=-1)

    B, K = case["B"], case["K"]
    tokens = torch.full((B, K + 1), -1, dtype=torch.int32, device=st["target"].device)
    accepted = torch.zeros(B, dtype=torch.int32, device=st["target"].device)
    drafts = st["tokens"].tolist()
    for b in range(B):
        p, q = probs(st["target"][b]), probs(st["draft"][b])
        a = 0
        while a < K and float(st["u"][b, a]) * float(q[a, drafts[b][a]]) < float(p[a, drafts[b][a]]):
            tokens[b, a] = drafts[b][a]
            a += 1
        rest = p[a] if a == K else (p[a] - q[a]).clamp(min=0)
        if not bool((rest > 0).any()):
            rest = p[a]
        tokens[b, a] = int(torch.argmax(rest / st["race"][b].double()))
        accepted[b] = a
    return tokens, accepted
