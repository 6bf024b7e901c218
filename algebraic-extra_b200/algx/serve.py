"""Answering with the language model: a paged cache, decoding, drafts and eviction.

``PagedCache`` owns the pages of all layers and hands them to sequences;
``Decoder`` runs ``algx.model.AlgebraicLM`` over it, prompts first and then one
or a few tokens at a time; ``generate`` and ``generate_with_draft`` sample from
it. They run the operators of ``algx.kernels.paged`` and ``algx.kernels.verify``
together as a serving loop uses them:

    dec = Decoder(model, batch=4, max_slots=2048)
    dec.prefill(prompts)                       # lists of token ids
    tokens = generate(dec, new_tokens=64)      # (4, 64) int32

The reference trains and evaluates only; this module has no counterpart there.

    python -m algx.serve --batch 4 --prompt 128 --new 64 [--draft-layers 2 --drafts 4] [--budget 256]

runs a randomly initialised model and prints tokens per second.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from . import rotary as R
from .kernels.flash import qknorm_flash_attention_packed
from .kernels.paged import cache_append, cache_evict, paged_attention
from .kernels.verify import verify_draft
from .layers import add_rms_norm, aluglu, rms_norm, swiglu

BF16 = torch.bfloat16


class PagedCache:
    """Key/value pages of every layer and the sequences' page table.

    ``k``, ``v`` (layers, pages, heads, page_size, 64) share one page numbering,
    so one table serves all layers. The free list is host state; ``table`` and
    ``lens`` are device tensors that the kernels read. ``reserve`` raises
    ``MemoryError`` when no page is left.
    """

    def __init__(self, layers: int, heads: int, batch: int, max_slots: int, *, page_size: int = 64,
                 pages: Optional[int] = None, dtype=BF16, device="cuda"):
        if batch < 1 or max_slots < 1:
            raise ValueError("batch and max_slots must be positive")
        self.page_size = int(page_size)
        self.max_pages = -(-int(max_slots) // self.page_size)
        pages = batch * self.max_pages if pages is None else int(pages)
        self.k = torch.zeros((layers, pages, heads, self.page_size, 64), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.zeros((batch, self.max_pages), dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free: List[int] = list(range(pages - 1, -1, -1))
        self.owned: List[List[int]] = [[] for _ in range(batch)]

    @property
    def slots(self) -> int:
        """Slots of one sequence's table."""
        return self.max_pages * self.page_size

    def _missing(self, need: Sequence[int]) -> int:
        """Pages that the free list lacks for ``need`` pages of each sequence."""
        return sum(max(0, n - len(o)) for n, o in zip(need, self.owned)) - len(self.free)

    def fits(self, slots: Sequence[int]) -> bool:
        """Whether ``reserve(slots)`` would find its slots and pages."""
        need = [-(-int(n) // self.page_size) for n in slots]
        return len(need) == len(self.owned) and max(need) <= self.max_pages and self._missing(need) <= 0

    def reserve(self, slots: Sequence[int]) -> None:
        """Give sequence b the pages of its first ``slots[b]`` slots."""
        need = [-(-int(n) // self.page_size) for n in slots]
        if len(need) != len(self.owned) or max(need) > self.max_pages:
            raise ValueError(f"at most {self.slots} slots for each of {len(self.owned)} sequences")
        if self._missing(need) > 0:
            raise MemoryError("no free pages")
        changed = False
        for n, own in zip(need, self.owned):
            while len(own) < n:
                own.append(self.free.pop())
                changed = True
        if changed:
            rows = [own + [0] * (self.max_pages - len(own)) for own in self.owned]
            self.table.copy_(torch.tensor(rows, dtype=torch.int32))

    def trim(self, slots: Sequence[int]) -> None:
        """Take back the pages beyond sequence b's first ``slots[b]`` slots."""
        for n, own in zip(slots, self.owned):
            while len(own) > -(-int(n) // self.page_size):
                self.free.append(own.pop())

    def release(self, b: int) -> None:
        """Take back every page of sequence b and forget its slots."""
        self.free.extend(reversed(self.owned[b]))
        self.owned[b] = []
        self.lens[b] = 0


class Decoder:
    """One model over its own paged cache, for ``batch`` sequences.

    ``max_slots`` bounds the cached tokens of a sequence, ``max_positions`` (default
    the same) their positions, which go on growing when slots are evicted.
    ``budget``: bring every layer's cache down to that many slots per head by
    accumulated attention weight whenever a sequence holds ``budget + slack``, and
    before a step that would otherwise find no slots or pages; the ``first`` first
    positions and the ``recent`` newest always stay (the weights that refused
    drafts gave stay counted).
    ``window``: a sliding window instead, with the ``first`` first slots visible.
    """

    def __init__(self, model, batch: int, max_slots: int, *, max_positions: Optional[int] = None,
                 page_size: int = 64, pages: Optional[int] = None, budget: Optional[int] = None, slack: int = 64,
                 first: int = 4, recent: Optional[int] = None, window: Optional[int] = None):
        cfg = model.cfg
        if budget is not None and window is not None:
            raise ValueError("eviction moves slots, which a window counts by: give budget or window")
        if budget is not None and not first < budget <= max_slots - slack:
            raise ValueError("budget must exceed first and leave slack below max_slots")
        if budget is not None and budget >= -(-max_slots // page_size) * page_size:
            raise ValueError("budget must leave slack: it fills every page of a sequence")
        dev = model.flat.data[True].device
        self.model, self.cfg, self.batch = model, cfg, int(batch)
        self.cache = PagedCache(cfg.n_layers, cfg.n_heads, batch, max_slots, page_size=page_size, pages=pages, device=dev)
        n = int(max_positions or max_slots)
        if cfg.pos == "rope":
            cos, sin = R.rope_table(64, n, cfg.rope_base, device=dev)
        else:
            cos, sin = R.cayley_table_geometric(64, n, cfg.rope_base, fraction=cfg.rope_fraction, device=dev)
        # the training forward rounds the tables to bfloat16 before it rotates
        self.rotary = tuple(t.to(BF16).float().contiguous() for t in (cos, sin))
        self.max_positions = n
        self.lens = [0] * batch       # cached slots, on the host too
        self.seen = [0] * batch       # tokens fed: the next position
        self.settled = [0] * batch    # first slots that an eviction left in no order of tokens
        self.positions = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.budget, self.slack, self.first = budget, int(slack), int(first)
        self.recent = min(recent if recent is not None else (budget or 0) // 4, (budget or 0) - first) if budget else 0
        self.window = window
        self.scores = self.slot_positions = None
        if budget is not None:
            shape = (cfg.n_layers, batch, cfg.n_heads, self.cache.slots)
            self.scores = torch.zeros(shape, dtype=torch.float32, device=dev)
            self.slot_positions = torch.full(shape, -1, dtype=torch.int32, device=dev)
        if cfg.sink == "const":
            self._sink = torch.full((cfg.n_heads,), cfg.sink_init, dtype=torch.float32, device=dev)
        self._scored = None           # logits (batch, rows, V) of the newest tokens, each sequence's newest row
        self.pending = None           # (batch,) the tokens that generate returned last, not fed yet

    @property
    def last(self):
        """(batch, V) float32 logits of every sequence's newest token; None before any, and where a rollback
        went behind the tokens of the last step."""
        if self._scored is None:
            return None
        logits, rows = self._scored
        if min(rows) == logits.shape[1] - 1:
            return logits[:, -1]
        return logits[torch.arange(self.batch, device=logits.device), torch.tensor(rows, device=logits.device)]

    # ------------------------------------------------------------ layers
    def _sink_of(self, i):
        if self.cfg.sink == "learned":
            return self.model.p(f"layers.{i}.sink").detach()
        return self._sink if self.cfg.sink == "const" else None

    def _layers(self, tokens, attend):
        """The model's blocks (model.py:184-200) with ``attend(i, qkv)`` for the attention; hidden (B, T, d)."""
        cfg, m = self.cfg, self.model
        B, T = tokens.shape
        p = m.p
        x = torch.nn.functional.embedding(tokens, p("embed")).to(BF16)
        x = rms_norm(x, p("embed_gain"), cfg.eps)
        h = rms_norm(x, p("layers.0.ln1"), cfg.eps)
        for i in range(cfg.n_layers):
            n = f"layers.{i}."
            qkv = m._mm(h, n + "w_qkv").view(B, T, 3, cfg.n_heads, 64)
            a = attend(i, qkv).view(B, T, cfg.d_model)
            x, h = add_rms_norm(x, m._mm(a, n + "w_o"), p(n + "ln2"), cfg.eps)
            gu = m._mm(h, n + "w_gu")
            act = swiglu(gu) if cfg.ffn == "swiglu" else aluglu(gu, cfg.alu_beta)
            gain = p(f"layers.{i + 1}.ln1") if i + 1 < cfg.n_layers else p("final_gain")
            x, h = add_rms_norm(x, m._mm(act, n + "w_d"), gain, cfg.eps)
        return h

    def _logits(self, h):
        """(rows, V) float32 logits of hidden rows against the tied embedding."""
        e = self.model.flat["embed"]
        hit = self.model._w16.get("embed")
        if hit is None or hit[0] != e._version:
            hit = self.model._w16["embed"] = (e._version, e.detach().to(BF16))
        return torch.mm(h.reshape(-1, h.shape[-1]), hit[1].t(), out_dtype=torch.float32)

    def _append(self, i, qkv, counts=None):
        B, T, _, H, D = qkv.shape
        n = f"layers.{i}."
        c = self.cache
        where = None if self.slot_positions is None else self.slot_positions[i]
        return cache_append(qkv.view(B, T, 3 * H, D), c.k[i], c.v[i], c.table, c.lens, self.model.p(n + "q_gain").detach(),
                            self.model.p(n + "k_gain").detach(), rotary=self.rotary, positions=self.positions,
                            counts=counts, slot_positions=where, eps=self.cfg.eps)

    # ------------------------------------------------------------ tokens
    @torch.no_grad()
    def step(self, tokens, idle: Sequence[int] = ()):
        """Feed ``tokens`` (B, T) int; float32 logits (B, T, V). The new slots stay until ``rollback``.

        The sequences named in ``idle`` sit the step out: they need no slots or
        positions and keep their weights; their rows of the result mean nothing.
        """
        cfg, c = self.cfg, self.cache
        B, T = tokens.shape
        idle = sorted(set(idle))
        by = [0 if b in idle else T for b in range(B)]
        if any(n and at + n > self.max_positions for n, at in zip(by, self.seen)):
            raise ValueError(f"positions end at {self.max_positions}")
        self.make_room(T, idle)
        c.reserve([n + t for n, t in zip(self.lens, by)])
        counts = torch.tensor(by, dtype=torch.int32, device=c.k.device) if idle else None
        after = c.lens + (T if counts is None else counts)
        known = self.last if idle else None
        held = self.scores[:, idle].clone() if self.scores is not None and idle else None

        def attend(i, qkv):
            q = self._append(i, qkv, counts)
            opts = dict(kind="asinh", n=cfg.attn_n, c=cfg.attn_c)
            if self.window is not None:
                opts.update(window=self.window, first=self.first)
            if self.scores is None:
                return paged_attention(q, c.k[i], c.v[i], c.table, after, self._sink_of(i), **opts)
            return paged_attention(q, c.k[i], c.v[i], c.table, after, self._sink_of(i), scores=self.scores[i], **opts)[0]

        logits = self._logits(self._layers(tokens, attend)).view(B, T, -1)
        if held is not None:
            self.scores[:, idle] = held
        self._advance(by)
        self._scored = logits, [T - 1] * B
        if idle:
            newest = logits[:, -1].clone()
            if known is not None:
                newest[idle] = known[idle]
            self._scored = None if known is None else (newest[:, None], [0] * B)
        return logits

    def make_room(self, tokens: int, idle: Sequence[int] = ()) -> None:
        """Evict now where ``tokens`` more tokens a sequence would find no slots or pages."""
        if self.budget is not None:
            if not self.cache.fits([n + (0 if b in idle else tokens) for b, n in enumerate(self.lens)]):
                self.evict(force=True)

    def _advance(self, by):
        self.pending = None
        self.lens = [n + t for n, t in zip(self.lens, by)]
        self.seen = [n + t for n, t in zip(self.seen, by)]
        self.cache.lens.copy_(torch.tensor(self.lens, dtype=torch.int32))
        self.positions.copy_(torch.tensor(self.seen, dtype=torch.int32))

    def rollback(self, drop):
        """Forget the newest ``drop[b]`` tokens of every sequence (refused drafts), fed since it was last evicted from."""
        if any(d < 0 or d > n for d, n in zip(drop, self.lens)):
            raise ValueError("cannot drop more tokens than are cached")
        if any(d > 0 and n - d < s for d, n, s in zip(drop, self.lens, self.settled)):
            raise ValueError("cannot drop tokens from before an eviction")
        self._advance([-int(d) for d in drop])
        self.cache.trim(self.lens)
        if self._scored is not None:
            logits, rows = self._scored
            rows = [r - int(d) for r, d in zip(rows, drop)]
            self._scored = (logits, rows) if min(rows) >= 0 else None

    @torch.no_grad()
    def prefill(self, prompts: Sequence[Sequence[int]]):
        """Feed one prompt (at least one token) per sequence into the empty cache; float32 logits (B, V) after them.

        Without a budget the training forward's tensor-core attention runs on the
        padded prompts (padding comes after the tokens, which do not see it) and
        ``cache_append`` stores their keys and values. With a budget the prompts go
        through the cache 64 tokens at a time, so that their weights are counted.
        """
        if len(prompts) != self.batch or any(len(p) == 0 for p in prompts):
            raise ValueError(f"one prompt of at least one token for each of {self.batch} sequences")
        if any(self.lens):
            raise ValueError("prefill needs an empty cache: use step")
        cfg, c, dev = self.cfg, self.cache, self.cache.k.device
        sizes = [len(p) for p in prompts]
        if self.budget is not None or self.window is not None:
            return self._prefill_steps(prompts, sizes)
        T = -(-max(sizes) // 128) * 128
        tokens = torch.zeros((self.batch, T), dtype=torch.int64)
        for b, p in enumerate(prompts):
            tokens[b, :len(p)] = torch.tensor(p)
        tokens = tokens.to(dev)
        if max(sizes) > self.max_positions:
            raise ValueError(f"positions end at {self.max_positions}")
        c.reserve(sizes)
        counts = torch.tensor(sizes, dtype=torch.int32, device=dev)
        # rotations of the padding's positions may lie beyond the tables; any will do
        rot = tuple(torch.cat([t, t[-1:].expand(max(0, T - t.shape[0]), -1)])[:T].contiguous() for t in self.rotary)

        def attend(i, qkv):
            n = f"layers.{i}."
            self._append(i, qkv, counts)
            return qknorm_flash_attention_packed(qkv, self.model.p(n + "q_gain"), self.model.p(n + "k_gain"),
                                                 self._sink_of(i), eps=cfg.eps, kind="asinh", n=cfg.attn_n, c=cfg.attn_c,
                                                 block=128, range_guard=True, rotary=rot)

        h = self._layers(tokens, attend)
        self._advance(sizes)
        last = self._logits(h[torch.arange(self.batch, device=dev), counts.long() - 1])
        self._scored = last[:, None], [0] * self.batch
        return last

    def _prefill_steps(self, prompts, sizes, chunk: int = 64):
        done = [0] * self.batch
        if self.budget is not None:
            chunk = min(chunk, self.cache.slots - self.budget)
        while any(d < n for d, n in zip(done, sizes)):
            # the sequences advance together, by what the one nearest its end still has
            left = [n - d for d, n in zip(done, sizes)]
            T = min(min(chunk, n) for n in left if n > 0)
            idle = [b for b, n in enumerate(left) if n == 0]
            rows = [[0] * T if b in idle else list(p[d:d + T]) for b, (p, d) in enumerate(zip(prompts, done))]
            self.step(torch.tensor(rows, device=self.cache.k.device), idle=idle)
            done = [d if b in idle else d + T for b, d in enumerate(done)]
            self.evict()
        return self.last

    @torch.no_grad()
    def evict(self, force: bool = False) -> bool:
        """Bring the cache down to its budget once a sequence holds ``slack`` more; whether it did."""
        if self.budget is None or (max(self.lens) < self.budget + (0 if force else self.slack)):
            return False
        c = self.cache
        for i in range(self.cfg.n_layers):
            _, scores, positions, _ = cache_evict(c.k[i], c.v[i], c.table, c.lens, self.scores[i],
                                                  self.slot_positions[i], budget=self.budget, first=self.first,
                                                  recent=self.recent)
            self.scores[i].copy_(scores)
            self.slot_positions[i].copy_(positions)
        self.settled = [self.budget if n > self.budget else s for n, s in zip(self.lens, self.settled)]
        self.lens = [min(n, self.budget) for n in self.lens]
        c.lens.copy_(torch.tensor(self.lens, dtype=torch.int32))
        c.trim(self.lens)
        return True


def head_options(cfg, temperature: float = 1.0) -> dict:
    """``verify_draft``'s options for a model's likelihood head."""
    if cfg.head == "ce":
        return dict(kind="ce", temperature=temperature)
    if temperature != 1.0:
        raise ValueError("temperature is for the ce kind")
    return dict(kind="alg_ce", n=cfg.head_n, c=cfg.head_c)


def _race(B, V, dev, generator):
    return torch.empty((B, V), dtype=torch.float32, device=dev).exponential_(generator=generator).clamp_min_(1e-30)


def sample(logits, cfg, generator=None, temperature: float = 1.0):
    """One token (B,) int32 from logits (B, V) under the model's head."""
    B, V = logits.shape
    none = torch.empty((B, 0), device=logits.device)
    out, _ = verify_draft(logits[:, None], none.to(torch.int32), None, none, _race(B, V, logits.device, generator),
                          **head_options(cfg, temperature))
    return out[:, 0]


@torch.no_grad()
def generate(dec: Decoder, new_tokens: int, *, generator=None, temperature: float = 1.0):
    """``new_tokens`` sampled tokens per sequence, (B, new_tokens) int32, after ``dec.prefill``.

    The last of them is not fed yet: it is ``dec.pending``, which the next call
    feeds first, so several calls go on where the one before ended. ``step`` and
    ``rollback`` forget it (a caller who steps feeds it with them).
    """
    if new_tokens < 1:
        return torch.empty((dec.batch, 0), dtype=torch.int32, device=dec.cache.k.device)
    if dec.pending is not None:
        dec.step(dec.pending[:, None])
        dec.evict()
    if dec.last is None:
        raise ValueError("the newest tokens' logits are not known: feed one with step" if any(dec.seen) else "prefill first")
    out = []
    for i in range(new_tokens):
        t = sample(dec.last, dec.cfg, generator, temperature)
        out.append(t)
        if i + 1 < new_tokens:
            dec.step(t[:, None])
            dec.evict()
    dec.pending = t
    return torch.stack(out, dim=1)


@torch.no_grad()
def generate_with_draft(dec: Decoder, draft: Decoder, new_tokens: int, *, drafts: int = 4, generator=None,
                        temperature: float = 1.0):
    """``generate`` with ``drafts`` tokens per round proposed by a smaller model; (tokens, accepted per round).

    Both decoders hold the same prompts, and the models share vocabulary and head.
    The tokens are distributed as ``generate``'s. Each round the draft model
    samples its tokens one by one, the target scores them and the one before in a
    single pass, and ``verify_draft`` accepts a prefix and draws the token after it.
    No sequence goes beyond its ``new_tokens``: drafts that would are not accepted,
    and sequences that are done sit out the others' rounds (with 0 accepted). A
    round takes slots and positions for ``drafts`` tokens that may be refused. As
    after ``generate`` the last tokens are both decoders' ``pending``.
    """
    a, b = dec.cfg, draft.cfg
    if (a.vocab_size, a.head, a.head_n, a.head_c) != (b.vocab_size, b.head, b.head_n, b.head_c):
        raise ValueError("the draft model needs the target's vocabulary and head")
    if not 1 <= drafts <= 31:
        raise ValueError("drafts must be from 1 to 31")
    if any(d.budget is not None and d.cache.slots - d.budget <= drafts for d in (dec, draft)):
        raise ValueError(f"a round needs room for {drafts + 1} tokens above the budget")
    if dec.pending is None or draft.pending is None:
        ready = dec.pending is draft.pending and dec.last is not None and draft.last is not None
    else:
        ready = torch.equal(dec.pending, draft.pending)
    if not ready or dec.seen != draft.seen:
        raise ValueError("prefill both decoders with the same prompts first")
    B, V, dev = dec.batch, a.vocab_size, dec.cache.k.device
    if new_tokens < 1:
        return torch.empty((B, 0), dtype=torch.int32, device=dev), []
    newest, out = dec.pending, [[] for _ in range(B)]
    if newest is None:
        newest = sample(dec.last, a, generator, temperature)
        out = [[t] for t in newest.tolist()]
    rounds = []
    while min(len(o) for o in out) < new_tokens:
        left = [new_tokens - len(o) for o in out]
        idle = [b for b, n in enumerate(left) if n == 0]
        tokens, logits = [newest], []
        draft.make_room(drafts + 1, idle)  # not between the steps: a rollback cannot go behind an eviction
        for _ in range(drafts):
            logits.append(draft.step(tokens[-1][:, None], idle)[:, 0])
            tokens.append(sample(logits[-1], a, generator, temperature))
        draft.step(tokens[-1][:, None], idle)  # its key and value, should all drafts be accepted
        fed = torch.stack(tokens, dim=1)
        scored = dec.step(fed, idle)
        u = torch.rand((B, drafts), device=dev, generator=generator)
        most = [min(drafts, max(0, n - 1)) for n in left]  # the token after them counts too
        counts = torch.tensor(most, dtype=torch.int32, device=dev) if min(most) < drafts else None
        got, accepted = verify_draft(scored, fed[:, 1:], torch.stack(logits, dim=1), u, _race(B, V, dev, generator),
                                     counts=counts, **head_options(a, temperature))
        took, rows = accepted.tolist(), got.tolist()
        drawn = got.gather(1, accepted[:, None].long())[:, 0]
        if idle:
            drawn[idle] = newest[idle]
        newest = drawn
        for b, (o, n, row) in enumerate(zip(out, took, rows)):
            if b not in idle:
                o.extend(row[:n + 1])
        for d in (dec, draft):
            d.rollback([0 if b in idle else drafts - n for b, n in enumerate(took)])
            d.evict()
        rounds.append([0 if b in idle else n for b, n in enumerate(took)])
    dec.pending = draft.pending = newest
    return torch.tensor(out, dtype=torch.int32, device=dev), rounds


def main(argv=None) -> None:
    """Generate with a randomly initialised model and print tokens per second."""
    import argparse
    import time

    from .model import AlgebraicLM, config_125m, config_algebraic_125m

    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--preset", choices=("standard", "algebraic"), default="standard")
    ap.add_argument("--layers", type=int, default=None, help="override n_layers")
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=128, help="tokens of each prompt")
    ap.add_argument("--new", type=int, default=64, help="tokens to generate per sequence")
    ap.add_argument("--budget", type=int, default=None, help="cache slots per head, by eviction")
    ap.add_argument("--window", type=int, default=None, help="sliding window, with 4 first tokens visible")
    ap.add_argument("--draft-layers", type=int, default=None, help="draft with a model of that many layers")
    ap.add_argument("--drafts", type=int, default=4, help="drafted tokens per round")
    args = ap.parse_args(argv)
    make = config_125m if args.preset == "standard" else config_algebraic_125m
    over = {} if args.layers is None else {"n_layers": args.layers}
    slots = args.prompt + args.new + args.drafts + 1
    opts = dict(batch=args.batch, max_slots=max(slots, (args.budget or 0) + 64), max_positions=slots,
                budget=args.budget, window=args.window)
    dec = Decoder(AlgebraicLM(make(**over)), **opts)
    gen = torch.Generator(device="cuda").manual_seed(0)
    prompts = torch.randint(0, dec.cfg.vocab_size, (args.batch, args.prompt)).tolist()
    dec.prefill(prompts)
    draft = None
    if args.draft_layers is not None:
        draft = Decoder(AlgebraicLM(make(n_layers=args.draft_layers)), **opts)
        draft.prefill(prompts)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    if draft is None:
        out, note = generate(dec, args.new, generator=gen), ""
    else:
        out, rounds = generate_with_draft(dec, draft, args.new, drafts=args.drafts, generator=gen)
        taken = sum(map(sum, rounds))  # each sequence's rounds gave its new tokens but the first, one beside the drafts
        played = args.batch * (args.new - 1) - taken
        note = f", {taken / max(1, played):.2f} of {args.drafts} drafts accepted a round"
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    print(f"{out.numel()} tokens in {dt * 1e3:.1f} ms, {out.numel() / dt:.0f} tokens/s{note}")


if __name__ == "__main__":
    main()
