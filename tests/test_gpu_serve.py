"""Serving loop on the GPU: decoding agrees with the training forward, drafts and eviction fit together."""

import pytest
import torch

from algx import _lib as L

pytestmark = pytest.mark.gpu


def small(preset="standard", layers=2, seed=3, **over):
    from algx.model import AlgebraicLM, config_125m, config_algebraic_125m
    make = config_125m if preset == "standard" else config_algebraic_125m
    cfg = make(vocab_size=512, d_model=128, n_heads=2, n_layers=layers, d_ff=256, seq_len=256, init_std=0.1, **over)
    return AlgebraicLM(cfg, seed=seed)


def full_logits(model, tokens):
    with torch.no_grad():
        h = model.forward_hidden(tokens)
        return h.float() @ model.flat["embed"].detach().to(torch.bfloat16).float().t()


def rel(a, b):
    return float(torch.linalg.norm(a.double() - b.double()) / torch.linalg.norm(b.double()))


@pytest.mark.parametrize("preset", ["standard", "algebraic"])
def test_decoding_matches_the_training_forward(preset):
    """Prompt and tokens one and several at a time, against one pass of the training forward over the
    same tokens: two blocks of bf16 activations, as in the model's own parity test (3e-2)."""
    from algx.serve import Decoder
    model = small(preset)
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 512, (3, 256), generator=g).cuda()
    want = full_logits(model, tokens)
    dec = Decoder(model, batch=3, max_slots=256)
    sizes = [100, 37, 1]
    got = dec.prefill([tokens[b, :n].tolist() for b, n in enumerate(sizes)])
    for b, n in enumerate(sizes):
        assert rel(got[b], want[b, n - 1]) < 3e-2
    for T in (1, 1, 5, 1):
        at = dec.lens
        step = torch.stack([tokens[b, at[b]:at[b] + T] for b in range(3)])
        logits = dec.step(step)
        for b in range(3):
            assert rel(logits[b], want[b, at[b]:at[b] + T]) < 3e-2
    assert dec.lens == [108, 45, 9] and dec.cache.lens.tolist() == dec.lens
    dec.rollback([3, 0, 8])
    at = dec.lens
    logits = dec.step(torch.stack([tokens[b, at[b]:at[b] + 2] for b in range(3)]))
    for b in range(3):
        assert rel(logits[b], want[b, at[b]:at[b] + 2]) < 3e-2
    assert L.device_error() == 0


def test_generation_with_and_without_drafts():
    from algx.serve import Decoder, generate, generate_with_draft
    prompts = [[1, 2, 3], [4, 5, 6, 7, 8]]
    gen = torch.Generator(device="cuda").manual_seed(0)
    dec = Decoder(small(), batch=2, max_slots=200)
    dec.prefill(prompts)
    out = generate(dec, 20, generator=gen)
    assert out.shape == (2, 20) and int(out.min()) >= 0 and int(out.max()) < 512
    assert dec.lens == [22, 24]

    # a draft model equal to the target is accepted but for roundings: its passes are one token wide
    target, draft = (Decoder(small(), batch=2, max_slots=200) for _ in range(2))
    for d in (target, draft):
        d.prefill(prompts)
    out, rounds = generate_with_draft(target, draft, 60, drafts=4, generator=gen)
    assert out.shape == (2, 60) and int(out.min()) >= 0 and int(out.max()) < 512
    assert sum(map(sum, rounds)) > 0.8 * 4 * 2 * len(rounds)
    assert target.lens == draft.lens and target.seen == draft.seen

    other = Decoder(small(layers=1, seed=9), batch=2, max_slots=200)
    fresh = Decoder(small(), batch=2, max_slots=200)
    for d in (other, fresh):
        d.prefill(prompts)
    out, rounds = generate_with_draft(fresh, other, 30, drafts=3, generator=gen)
    assert out.shape == (2, 30) and all(0 <= n <= 3 for r in rounds for n in r)
    assert L.device_error() == 0


def test_eviction_bounds_the_cache_and_keeps_its_heavy_slots():
    from algx.serve import Decoder, generate
    model = small("algebraic")
    gen = torch.Generator(device="cuda").manual_seed(0)
    prompts = torch.randint(0, 512, (2, 90), generator=torch.Generator().manual_seed(2)).tolist()
    dec = Decoder(model, batch=2, max_slots=160, max_positions=400, budget=64, slack=16, first=4, recent=16, page_size=16)
    dec.prefill(prompts)
    generate(dec, 150, generator=gen)
    assert max(dec.lens) < 64 + 16 + 1 and dec.seen == [239, 239]
    assert all(len(o) <= -(-(64 + 16 + 1) // 16) for o in dec.cache.owned)
    dec.evict(force=True)
    for b in range(2):
        n = dec.lens[b]
        pos = dec.slot_positions[:, b, :, :n]
        for first in range(4):
            assert bool((pos == first).any(dim=-1).all())
        for recent in range(239 - 16, 239):
            assert bool((pos == recent).any(dim=-1).all())
        assert bool((dec.slot_positions[:, b, :, n:] == -1).all()) and bool((dec.scores[:, b, :, n:] == 0).all())
    assert L.device_error() == 0


def test_an_ample_budget_and_window_change_nothing():
    from algx.serve import Decoder
    model = small()
    tokens = torch.randint(0, 512, (1, 80), generator=torch.Generator().manual_seed(4)).cuda()
    want = full_logits(model, torch.nn.functional.pad(tokens, (0, 176)))[:, 70:80]
    for opts in (dict(budget=120, slack=16), dict(window=500)):
        dec = Decoder(model, batch=1, max_slots=160, **opts)
        dec.prefill([tokens[0, :70].tolist()])
        assert rel(dec.step(tokens[:, 70:80]), want) < 3e-2


def test_decoder_refuses():
    from algx.serve import Decoder, generate
    model = small(layers=1)
    with pytest.raises(ValueError, match="budget or window"):
        Decoder(model, batch=1, max_slots=64, budget=32, window=16)
    with pytest.raises(ValueError, match="leave slack"):
        Decoder(model, batch=1, max_slots=64, budget=32, slack=64)
    dec = Decoder(model, batch=1, max_slots=64)
    with pytest.raises(ValueError, match="prefill first"):
        generate(dec, 4)
    with pytest.raises(ValueError, match="at least one token"):
        dec.prefill([[]])
    dec.prefill([[1, 2]])
    with pytest.raises(ValueError, match="empty cache"):
        dec.prefill([[1, 2]])
    with pytest.raises(ValueError, match="cannot drop"):
        dec.rollback([3])
    with pytest.raises(ValueError, match="positions end"):
        dec.step(torch.zeros((1, 63), dtype=torch.int64, device="cuda"))


def test_command_line(capsys):
    from algx.serve import main
    main(["--layers", "1", "--batch", "2", "--prompt", "20", "--new", "8", "--draft-layers", "1", "--drafts", "2"])
    assert "tokens/s" in capsys.readouterr().out


def test_drafting_with_another_model_in_no_more_room_than_it_needs(capsys):
    """Sequences accept differently; the command line's sizes leave one round of drafts beyond the new tokens."""
    from algx.serve import Decoder, generate_with_draft, main
    prompts = torch.randint(0, 512, (4, 16), generator=torch.Generator().manual_seed(6)).tolist()
    target, draft = (Decoder(small(layers=n, seed=n), batch=4, max_slots=16 + 48 + 5) for n in (2, 1))
    for d in (target, draft):
        d.prefill(prompts)
    out, rounds = generate_with_draft(target, draft, 48, generator=torch.Generator(device="cuda").manual_seed(1))
    assert out.shape == (4, 48) and target.lens == draft.lens == [16 + 47] * 4
    assert len({sum(r[b] for r in rounds) for b in range(4)}) > 1
    full = torch.cat([torch.tensor(prompts).cuda(), out[:, :-1]], dim=1)
    assert rel(target.step(out[:, -1:])[:, 0], full_logits(target.model, torch.nn.functional.pad(
        torch.cat([full, out[:, -1:]], dim=1), (0, 192)))[:, 63]) < 3e-2
    main(["--layers", "2", "--batch", "4", "--prompt", "20", "--new", "40", "--draft-layers", "1"])
    assert "tokens/s" in capsys.readouterr().out and L.device_error() == 0


@pytest.mark.parametrize("opts", [dict(), dict(budget=100, slack=16), dict(window=20)])
def test_idle_sequences_stay_as_they_are(opts):
    from algx.serve import Decoder
    model = small()
    tokens = torch.randint(0, 512, (2, 60), generator=torch.Generator().manual_seed(7)).cuda()
    a, b = (Decoder(model, batch=2, max_slots=128, **opts) for _ in range(2))
    for d in (a, b):
        d.prefill([r[:30].tolist() for r in tokens])
    a.step(tokens[:, 30:33])
    b.step(tokens[:, 30:33])
    last = b.last[1].clone()
    mixed = torch.stack([tokens[0, 33:38], torch.zeros_like(tokens[1, 33:38])])
    got, want = b.step(mixed, idle=[1])[0], a.step(tokens[:, 33:38])[0]
    assert torch.equal(got, want) and torch.equal(b.last[1], last) and b.lens == [38, 33]
    a.rollback([0, 5])
    if a.scores is not None:
        assert torch.equal(b.scores[:, 0], a.scores[:, 0])
        assert bool((b.scores[:, 1, :, :33].sum(-1) < a.scores[:, 1, :, :33].sum(-1)).all())
    assert torch.equal(b.step(tokens[:, 38:40])[0], a.step(tokens[:, 38:40])[0]) and L.device_error() == 0
