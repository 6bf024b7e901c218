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
from algx.serve import Decoder, generate, generate_with_draft
from oracle import serving_math as O

V = 23


def logits_of(held, like, seed):
    """Logits after the cached (position, token) pairs ``held``; ``like`` of them is the same for every seed."""
    g = torch.Generator().manual_seed(hash(tuple(held)) % 2 ** 62)
    common = torch.randn(V, generator=g)
    own = torch.randn(V, generator=g.manual_seed(hash((seed, tuple(held))) % 2 ** 62))
    return 2 * (like * common + (1 - like) * own)


class Toy(Decoder):
    def __init__(self, batch, max_slots, *, like=1.0, seed=0, **kw):
        cfg = config_125m(vocab_size=V, d_model=64, n_heads=1, n_layers=1, d_ff=64)
        model = SimpleNamespace(cfg=cfg, flat=SimpleNamespace(data={True: torch.zeros(1)}), p=lambda name: torch.zeros(1))
        super().__init__(model, batch, max_slots, **kw)
        self.cache.k = self.cache.k.float()  # (position, token) of every slot
        self.toy = like, seed

    def held(self, b):
        """(position, token) of the cached slots of sequence b, by position."""
        return sorted(pairs(self.cache.k[0], self.cache.table[b], int(self.cache.lens[b])))

    def tokens(self, b):
        held = self.held(b)
        assert [p for p, _ in held] == list(range(self.seen[b]))
        return [t for _, t in held]

    def logits_of(self, held):
        return logits_of(held, *self.toy)

    def _sink_of(self, i):
        return self.toy

    def _layers(self, tokens, attend):
        B, T = tokens.shape
        return attend(0, tokens[:, :, None, None, None].expand(B, T, 3, 1, 64).float())

    def _logits(self, h):
        return h.reshape(-1, 64)[:, :V]


def pairs(k, table, count):
    return [(int(r[0]), int(r[1])) for r in O.slots_of(k, table, count, 0)]


def append(qkv, k, v, table, lens, gain_q, gain_k, *, rotary, positions, counts=None, slot_positions=None, eps):
    """``cache_append``: tokens and positions in place of keys."""
    B, T, size = *qkv.shape[:2], k.shape[2]
    for b in range(B):
        for t in range(T if counts is None else int(counts[b])):
            s, at = int(lens[b]) + t, int(positions[b]) + t
            assert at < rotary[0].shape[0]
            k[int(table[b, s // size]), 0, s % size, :2] = torch.tensor([float(at), float(qkv[b, t, 0, 0])])
            if slot_positions is not None:
                slot_positions[b, 0, s] = at
    return qkv[:, :, :1]


def attention(q, k, v, table, lens, sink, *, scores=None, **kw):
    """``paged_attention``: the logits of what each query sees in place of its output."""
    B, T = q.shape[:2]
    out = torch.zeros((B, T, 1, 64))
    for b in range(B):
        n = int(lens[b])
        held = pairs(k, table[b], n)
        if scores is not None:
            scores[b, 0, max(0, n - T):] = 0.0
        for t in range(T):
            seen = held[:max(0, n - T + t + 1)]
            out[b, t, 0, :V] = logits_of(sorted(seen), *sink)
            if scores is not None:
                scores[b, 0, :len(seen)] += torch.tensor([float(1 + (7 * p + 3 * len(seen)) % 5) for p, _ in seen])
    return out if scores is None else (out, scores)


def prompt_attention(qkv, gain_q, gain_k, sink, **kw):
    B, T = qkv.shape[:2]
    out = torch.zeros((B, T, 1, 64))
    for b in range(B):
        row = [(t, int(qkv[b, t, 0, 0, 0])) for t in range(T)]
        for t in range(T):
            out[b, t, 0, :V] = logits_of(row[:t + 1], *sink)
    return out


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
    monkeypatch.setattr(serve, "cache_append", append)
    monkeypatch.setattr(serve, "paged_attention", attention)
    monkeypatch.setattr(serve, "qknorm_flash_attention_packed", prompt_attention)


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


def drafting(n_new, drafts=4, like=0.6, prompts=PROMPTS, extra=0, **kw):
    """A target and a draft decoder with no slot to spare: what the longest prompt, the new tokens and one round of
    drafts take."""
    slots = max(map(len, prompts)) + n_new + drafts + 1
    kw = dict(max_slots=slots, max_positions=slots, page_size=16, prompts=prompts, **kw)
    return toy(like=like, seed=1, **kw), toy(like=like, seed=2, **kw)


@pytest.mark.parametrize("like", [0.3, 0.6, 0.9, 1.0])
@pytest.mark.parametrize("drafts", [1, 4, 7])
def test_drafting_ends_every_sequence_at_its_last_token(drafts, like):
    """Sequences of different acceptance: those that are done wait for the others, within slots and positions that
    hold nothing beyond one round."""
    n_new = 30
    dec, draft = drafting(n_new, drafts, like)
    out, rounds = generate_with_draft(dec, draft, n_new, drafts=drafts, generator=gen(5))
    assert out.shape == (3, n_new) and out.dtype == torch.int32
    for d in (dec, draft):
        assert [d.tokens(b) for b in range(3)] == [p + out[b, :-1].tolist() for b, p in enumerate(PROMPTS)]
        assert torch.equal(d.pending, out[:, -1])
    assert all(0 <= n <= drafts for r in rounds for n in r)
    if like == 1.0:  # equal models: every draft is accepted
        assert sum(r[0] for r in rounds) == n_new - 1 - len(rounds)


def test_drafting_goes_on_after_drafting_and_into_plain_generation():
    dec, draft = drafting(40)
    g = gen(6)
    out = [generate_with_draft(dec, draft, n, generator=g)[0] for n in (9, 1, 12)]
    out.append(generate(dec, 5, generator=g))
    out = torch.cat(out, dim=1)
    assert [dec.tokens(b) for b in range(3)] == [p + out[b, :-1].tolist() for b, p in enumerate(PROMPTS)]
    with pytest.raises(ValueError, match="same prompts"):
        generate_with_draft(dec, draft, 3, generator=g)  # the draft model has not seen the last five


def test_drafting_refuses_decoders_that_stand_at_different_tokens():
    dec, draft = drafting(40)
    generate(dec, 3, generator=gen(7))
    generate(draft, 3, generator=gen(8))
    assert dec.seen == draft.seen and not torch.equal(dec.pending, draft.pending)
    with pytest.raises(ValueError, match="same prompts"):
        generate_with_draft(dec, draft, 3)
    dec, draft = drafting(40)
    for n in (0, 32):
        with pytest.raises(ValueError, match="drafts"):
            generate_with_draft(dec, draft, 3, drafts=n)
    assert generate_with_draft(dec, draft, 0)[0].shape == (3, 0)


def test_sequences_that_wait_keep_their_weights():
    """Under a budget the accumulated weights of a finished sequence stay as they are while the others go on."""
    prompts = [[1, 2, 3], [4, 5, 6]]
    kw = dict(max_slots=96, max_positions=96, page_size=16, budget=80, slack=8, prompts=prompts)
    dec, alone = toy(**kw), toy(**kw)
    fed = torch.randint(0, V, (2, 6), generator=gen(9))
    dec.step(fed[:, :3], idle=[])
    before = dec.scores[:, 1].clone(), dec.last[1].clone()
    dec.step(fed[:, 3:], idle=[1])
    assert dec.lens == [9, 6] and dec.seen == [9, 6] and dec.cache.lens.tolist() == [9, 6]
    assert torch.equal(dec.scores[:, 1], before[0]) and torch.equal(dec.last[1], before[1])
    alone.step(fed[:, :3])
    alone.step(fed[:, 3:])
    assert torch.equal(dec.scores[:, 0], alone.scores[:, 0]) and torch.equal(dec.last[0], alone.last[0])
    assert dec.tokens(1) == prompts[1] + fed[1, :3].tolist()


@pytest.mark.parametrize("page_size,max_slots,budget,slack,sizes", [
    (64, 320, 256, 64, [40, 500]),
    (16, 164, 100, 64, [400]),
    (64, 2112, 2048, 64, [2300, 30]),
    (16, 48, 40, 8, [200, 7, 90]),   # less slack than a chunk of the prompt
    (16, 41, 40, 1, [60]),
])
def test_a_budget_runs_in_the_least_slots(page_size, max_slots, budget, slack, sizes):
    prompts = [torch.randint(0, V, (n,), generator=gen(n)).tolist() for n in sizes]
    dec = toy(max_slots, page_size, prompts, max_positions=3000, budget=budget, slack=slack, first=2, recent=5)
    assert dec.seen == sizes and max(dec.lens) < budget + slack
    assert torch.equal(dec.last, newest(dec)) or max(sizes) > budget  # an eviction forgets what the logits had seen
    for b, p in enumerate(prompts):
        held = dec.held(b)
        assert len(held) == min(len(p), dec.lens[b]) and all(p[at] == t for at, t in held)
        assert {at for at, _ in held} >= set(range(min(2, len(p)))) | set(range(max(0, len(p) - 5), len(p)))
    generate(dec, 2 * slack + 3, generator=gen(10))
    assert max(dec.lens) < budget + slack


def test_drafting_under_a_budget_in_the_least_slots():
    """Rounds of five tokens meet the end of the tables at every distance."""
    prompts = [torch.randint(0, V, (n,), generator=gen(n)).tolist() for n in (40, 11)]
    kw = dict(prompts=prompts, max_slots=48, max_positions=400, page_size=16, budget=40, slack=8, first=2, recent=9)
    dec, draft = toy(like=0.7, seed=1, **kw), toy(like=0.7, seed=2, **kw)
    out, _ = generate_with_draft(dec, draft, 90, generator=gen(11))
    for d in (dec, draft):
        for b, p in enumerate(prompts):
            fed = p + out[b, :-1].tolist()
            assert d.seen[b] == len(fed) and all(fed[at] == t for at, t in d.held(b))
            assert {at for at, _ in d.held(b)} >= {0, 1} | set(range(len(fed) - 9, len(fed)))
    with pytest.raises(ValueError, match="room for 9 tokens"):
        generate_with_draft(dec, draft, 10, drafts=8)


def test_an_eviction_makes_room_when_pages_run_out():
    """Fewer pages than the tables could name: what the budget frees is taken before giving up."""
    prompts = [torch.randint(0, V, (n,), generator=gen(n)).tolist() for n in (44, 44)]
    dec = toy(64, 16, prompts, max_positions=200, budget=32, slack=30, first=2, recent=5, pages=6)
    generate(dec, 30, generator=gen(12))
    assert dec.seen == [73, 73]


def test_a_budget_needs_a_slot_beside_it():
    with pytest.raises(ValueError, match="leave slack"):
        toy(48, budget=48, slack=0)
    assert toy(40, budget=40, slack=0, first=2, recent=4).cache.slots == 48  # the last page's


def test_a_rollback_does_not_go_behind_an_eviction():
    """Evicted sequences hold their slots in no order of tokens; the others' still are."""
    prompts = [torch.randint(0, V, (n,), generator=gen(n)).tolist() for n in (36, 9)]
    dec = toy(64, 16, prompts, max_positions=200, budget=30, slack=10, first=2, recent=5)
    assert dec.evict(force=True) and dec.lens == [30, 9]
    dec.step(torch.zeros((2, 3), dtype=torch.int64))
    before = dec.held(0), dec.held(1)
    with pytest.raises(ValueError, match="cannot drop tokens from before an eviction"):
        dec.rollback([4, 0])
    assert (dec.held(0), dec.held(1)) == before and dec.lens == [33, 12]
    dec.rollback([3, 8])
    assert dec.lens == [30, 4] and dec.tokens(1) == prompts[1][:4]
    assert max(p for p, _ in dec.held(0)) == 35
    with pytest.raises(ValueError, match="cannot drop more tokens"):
        dec.rollback([0, 5])
