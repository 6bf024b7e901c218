"""The serving loop's own bookkeeping on CPU, with stand-ins for the kernels.

``Toy`` is a ``Decoder`` whose model is a table: the logits of a token are drawn from
a generator seeded by everything that the sequence's cache then holds, read back through
its page table. A token that is missing, doubled or left over after a rollback changes them.
Append, eviction and verification are the 64-bit restatements.
"""

from types import SimpleNamespace

import pytest
import torch

from algx import serve
from algx.model import config_125m
from algx.serve import Decoder, generate
from oracle import serving_math as O

V = 23


class Toy(Decoder):
    def __init__(self, batch, max_slots, *, like=1.0, seed=0, **kw):
        cfg = config_125m(vocab_size=V, d_model=64, n_heads=1, n_layers=1, d_ff=64)
        super().__init__(SimpleNamespace(cfg=cfg, flat=SimpleNamespace(data={True: torch.zeros(1)})), batch, max_slots, **kw)
        self.cache.k = self.cache.k.float()  # (position, token) of every slot
        self.like, self.seed = like, seed    # how much of the logits all toys share

    def held(self, b):
        """(position, token) of the cached slots of sequence b, by position."""
        rows = O.slots_of(self.cache.k[0], self.cache.table[b], int(self.cache.lens[b]), 0)
        return sorted((int(r[0]), int(r[1])) for r in rows)

    def tokens(self, b):
        held = self.held(b)
        assert [p for p, _ in held] == list(range(self.seen[b]))
        return [t for _, t in held]

    def logits_of(self, held):
        g = torch.Generator().manual_seed(hash(tuple(held)) % 2 ** 62)
        common = torch.randn(V, generator=g)
        own = torch.randn(V, generator=g.manual_seed(hash((self.seed, tuple(held))) % 2 ** 62))
        return 2 * (self.like * common + (1 - self.like) * own)

    def _layers(self, tokens, attend):
        c, size = self.cache, self.cache.page_size
        B, T = tokens.shape
        out = torch.zeros((B, T, V))
        for b in range(B):
            n, start = int(c.lens[b]), int(self.positions[b])
            slots = [(int(c.table[b, s // size]), s % size) for s in range(n) if s // size < len(c.owned[b])]
            held = [tuple(int(x) for x in c.k[0, p, 0, r, :2]) for p, r in slots]
            for t in range(T):
                s = n + t
                if s // size < len(c.owned[b]):
                    page, row = c.owned[b][s // size], s % size
                    c.k[0, page, 0, row, 0], c.k[0, page, 0, row, 1] = start + t, int(tokens[b, t])
                    if self.scores is not None:
                        self.slot_positions[0, b, 0, s] = start + t
                        self.scores[0, b, 0, s] = 0.0
                        for i, (p, _) in enumerate(held):
                            self.scores[0, b, 0, i] += 1 + (7 * p + 3 * start + t) % 5
                held.append((start + t, int(tokens[b, t])))
                out[b, t] = self.logits_of(sorted(held))
        return out

    def _logits(self, h):
        return h.reshape(-1, V)


def evict(k, v, table, lens, scores, positions, *, budget, first=0, recent=0):
    """``cache_evict`` for one head."""
    new_scores, new_positions = torch.zeros_like(scores), torch.full_like(positions, -1)
    size, old = k.shape[2], k.clone()
    for b in range(len(lens)):
        plan = O.evict_plan(scores[b, 0], positions[b, 0], int(lens[b]), budget, first, recent)
        for to, of in enumerate(plan):
            new_scores[b, 0, to], new_positions[b, 0, to] = scores[b, 0, of], positions[b, 0, of]
            k[int(table[b, to // size]), 0, to % size] = old[int(table[b, of // size]), 0, of % size]
    return lens.clamp(max=budget), new_scores, new_positions, None


def verify(target, tokens, draft, u, race, *, counts=None, **kw):
    out, accepted = O.verify_draft(target, tokens, draft, u, race, counts=None if counts is None else counts.tolist(), **kw)
    return torch.tensor(out, dtype=torch.int32), torch.tensor(accepted, dtype=torch.int32)


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    monkeypatch.setattr(serve, "cache_evict", evict)
    monkeypatch.setattr(serve, "verify_draft", verify)


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


PROMPTS = [[3, 1, 4, 1, 5], [9, 2], [6, 5, 3, 5, 8, 9, 7, 9, 3]]


def toy(max_slots=64, page_size=16, prompts=PROMPTS, **kw):
    dec = Toy(len(prompts), max_slots, page_size=page_size, **kw)
    dec.prefill(prompts)
    return dec


def newest(dec):
    return torch.stack([dec.logits_of(dec.held(b)) for b in range(dec.batch)])


def test_the_newest_logits_follow_prompts_and_steps():
    dec = toy()
    assert [dec.tokens(b) for b in range(3)] == PROMPTS
    assert torch.equal(dec.last, newest(dec))
    dec.step(torch.randint(0, V, (3, 4), generator=gen()))
    assert torch.equal(dec.last, newest(dec)) and dec.lens == [9, 6, 13]


@pytest.mark.parametrize("drop", [[3, 0, 1], [1, 1, 1], [0, 0, 0]])
def test_the_newest_logits_after_a_rollback_are_those_of_the_tokens_left(drop):
    dec = toy()
    dec.step(torch.randint(0, V, (3, 4), generator=gen()))
    dec.rollback(drop)
    assert torch.equal(dec.last, newest(dec))
    dec.rollback([0, 0, 1] if max(drop) < 3 else [0, 0, 0])
    assert torch.equal(dec.last, newest(dec))


def test_logits_of_tokens_before_the_newest_step_are_not_known():
    dec = toy()
    dec.step(torch.zeros((3, 1), dtype=torch.int64))
    dec.step(torch.zeros((3, 2), dtype=torch.int64))
    dec.rollback([1, 2, 0])
    assert dec.last is None
    with pytest.raises(ValueError, match="not known"):
        generate(dec, 2, generator=gen())
    dec.step(torch.zeros((3, 1), dtype=torch.int64))
    assert torch.equal(dec.last, newest(dec))
    assert generate(dec, 2, generator=gen()).shape == (3, 2)


def test_generating_in_pieces_is_generating_at_once():
    """The token that a call returned last is fed before the next one is drawn."""
    whole = toy()
    want = generate(whole, 11, generator=gen(1))
    dec, g = toy(), gen(1)
    parts = [generate(dec, n, generator=g) for n in (4, 1, 0, 6)]
    assert torch.equal(torch.cat(parts, dim=1), want) and want.shape == (3, 11)
    for d in (whole, dec):
        assert [d.tokens(b) for b in range(3)] == [p + want[b, :-1].tolist() for b, p in enumerate(PROMPTS)]
        assert torch.equal(d.pending, want[:, -1])


def test_a_token_not_fed_yet_is_forgotten_by_steps_and_rollbacks():
    dec = toy()
    out = generate(dec, 3, generator=gen(2))
    dec.step(torch.full((3, 1), 7))  # the caller goes on with a token of its own
    assert dec.pending is None and torch.equal(dec.last, newest(dec))
    generate(dec, 2, generator=gen(3))
    dec.rollback([1, 0, 0])
    assert dec.pending is None
    dec.step(torch.full((3, 1), 8))
    assert dec.tokens(1)[:-2] == PROMPTS[1] + out[1, :2].tolist() + [7]
    assert generate(dec, 0).shape == (3, 0)


def test_pieces_under_a_budget():
    kw = dict(max_slots=48, max_positions=200, budget=24, slack=8, first=2, recent=6)
    whole = toy(**kw)
    want = generate(whole, 40, generator=gen(4))
    dec, g = toy(**kw), gen(4)
    assert torch.equal(torch.cat([generate(dec, n, generator=g) for n in (13, 20, 7)], dim=1), want)
    assert dec.lens == whole.lens and [dec.held(b) for b in range(3)] == [whole.held(b) for b in range(3)]
