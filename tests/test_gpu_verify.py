"""Draft verification against its 64-bit restatement (oracle/serving_math.py)."""

import math

import pytest
import torch

from algx import _lib as L
from algx.kernels.verify import verify_draft
from oracle import serving_math as O

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
BAD_LABEL = 4


def inputs(B, K, V, dtype, kind, c, seed, spread=0.7, n=8):
    """Drafts are drawn from the draft model's own probabilities, as the operator's contract says."""
    g = torch.Generator().manual_seed(seed)
    unit = c if kind == "alg_ce" else 1.0
    base = 2 * torch.randn((B, K + 1, V), generator=g)
    draft = base[:, :K] + spread * torch.randn((B, K, V), generator=g)
    target, draft = (base * unit).to(dtype), (draft * unit).to(dtype)
    logq = draft.float() if kind == "ce" else n * torch.asinh(draft.float() / c)
    tokens = torch.empty((B, 0), dtype=torch.int32)
    if K:
        tokens = torch.multinomial(torch.softmax(logq, -1).reshape(-1, V), 1, generator=g).reshape(B, K).to(torch.int32)
    u = torch.rand((B, K), generator=g)
    race = (-torch.log1p(-torch.rand((B, V), generator=g))).clamp_min(1e-30)
    return target, tokens, draft, u, race


def check(target, tokens, draft, u, race, counts=None, **kw):
    want, acc = O.verify_draft(target, tokens, draft, u, race, counts=counts, **kw)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    cd = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
    out, got = verify_draft(dev(target), dev(tokens), dev(draft), dev(u), dev(race), counts=cd, **kw)
    assert out.dtype == got.dtype == torch.int32
    assert got.tolist() == acc and out.tolist() == want


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind,n,c", [("ce", 16, 16.0), ("alg_ce", 8, 2.0), ("alg_ce", 32, 16.0)])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (2, 4, 7), (3, 3, 257), (5, 7, 1000), (2, 31, 130), (2, 4, 50304),
                                   (1, 5, 32001), (300, 2, 33)])
def test_verify(B, K, V, kind, n, c, dtype):
    check(*inputs(B, K, V, dtype, kind, c, 60 + V, n=n), kind=kind, n=n, c=c)


@pytest.mark.parametrize("kind", ["ce", "alg_ce"])
@pytest.mark.parametrize("B,K,V", [(1, 3, 50304), (3, 31, 6241), (3, 31, 6242), (9, 1, 3968)])
def test_few_sequences_over_either_size_of_cluster(B, K, V, kind):
    """The number of CTAs a sequence depends on how much there is to read."""
    check(*inputs(B, K, V, F32, kind, 2.0, 20 + K, n=8), kind=kind, n=8, c=2.0)


@pytest.mark.parametrize("kind", ["ce", "alg_ce"])
def test_sampling_without_drafts(kind):
    target, tokens, _, u, race = inputs(6, 0, 999, F32, kind, 2.0, 1)
    check(target, tokens, None, u, race, kind=kind, n=8, c=2.0)


def test_certain_proposals_ragged_counts_and_temperature():
    target, tokens, draft, u, race = inputs(6, 5, 300, BF16, "ce", 1.0, 2)
    tokens = target[:, :5].float().argmax(-1).to(torch.int32)
    check(target, tokens, None, u * 0.5, race)
    check(target, tokens, draft, u, race, counts=[0, 1, 2, 3, 4, 5])
    check(target, tokens, draft, u, race, counts=[5, 0, 99, -3, 1, 1])  # cut to 0 .. K
    for t in (0.25, 3.0):
        check(target, tokens, draft, u, race, temperature=t)


def test_equal_models_accept_everything():
    target, tokens, _, u, race = inputs(8, 6, 5000, BF16, "ce", 1.0, 3)
    draft = target[:, :6].clone()
    tokens = torch.multinomial(torch.softmax(draft.float(), -1).reshape(-1, 5000), 1).reshape(8, 6).to(torch.int32)
    check(target, tokens, draft, u, race)
    out, acc = verify_draft(target.cuda(), tokens.cuda(), draft.cuda(), u.cuda(), race.cuda())
    assert acc.tolist() == [6] * 8


def test_nothing_left_of_the_residual_falls_back_to_p():
    """u = 1 refuses a draft of equal models, whose residual is zero everywhere."""
    target, tokens, _, u, race = inputs(2, 2, 500, F32, "ce", 1.0, 4)
    check(target, tokens, target[:, :2].clone(), torch.ones_like(u), race)


@pytest.mark.parametrize("kind", ["ce", "alg_ce"])
def test_masked_and_odd_logits(kind):
    target, tokens, draft, u, race = inputs(4, 3, 600, F32, kind, 2.0, 5)
    target[:, :, 100:] = -math.inf
    draft[:, :, ::2] = -math.inf
    target[1, :, 7] = math.nan
    target[2] = -math.inf              # no probability anywhere: token 0
    target[3, :, 50] = 1e4 if kind == "ce" else 1e15  # one token has it all
    tokens[3] = 50
    check(target, tokens, draft, u, race, kind=kind, n=16, c=2.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K", [0, 2])
def test_rows_of_the_lowest_finite_logits(K, dtype):
    """Masks of the type's lowest value: beside other logits they have no probability, alone they are as likely as
    each other."""
    low = torch.finfo(dtype).min
    target, tokens, draft, u, race = inputs(6, K, 700, dtype, "ce", 1.0, 12)
    target[0] = low
    target[1, :, 40:] = low
    target[2, :, :699] = low
    target[3, :, ::2], target[3, :, 1::2] = low, -math.inf
    target[4] = -3e38 if dtype == F32 else low
    draft[:4:2] = low
    draft[5, :, 5:] = low
    check(target, tokens, draft if K else None, u, race)
    check(target, tokens, draft if K else None, u, race, temperature=1e38)


def test_draft_tokens_outside_the_vocabulary_are_refused():
    target, tokens, draft, u, race = inputs(3, 3, 400, BF16, "ce", 1.0, 6)
    tokens[0, 0], tokens[1, 2] = -1, 400
    L.device_error()
    check(target, tokens, draft, u, race)
    assert L.device_error() & BAD_LABEL


def test_strided_logits_and_no_sequences():
    target, tokens, draft, u, race = inputs(3, 2, 129, BF16, "ce", 1.0, 7)
    wide = torch.zeros((3, 3, 200), dtype=BF16, device="cuda")
    wide[..., :129] = target.cuda()
    rest = [t.cuda() for t in (tokens, draft, u, race)]
    a = verify_draft(wide[..., :129], *rest)
    b = verify_draft(target.cuda(), *rest)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    out, acc = verify_draft(wide[:0, :, :129], *(t[:0] for t in rest))
    assert out.shape == (0, 3) and acc.shape == (0,)


def test_tokens_have_the_target_distribution():
    """Over many seeds the first token is distributed as p, whatever the draft: each frequency
    within six standard deviations of its probability."""
    V, B = 8, 40000
    g = torch.Generator().manual_seed(8)
    p, q = torch.randn(V, generator=g), torch.randn(V, generator=g)
    target = p.expand(B, 2, V).contiguous().cuda()
    draft = q.expand(B, 1, V).contiguous().cuda()
    tokens = torch.multinomial(torch.softmax(q, -1), B, replacement=True, generator=g).reshape(B, 1).to(torch.int32)
    u = torch.rand((B, 1), generator=g)
    race = torch.empty((B, V)).exponential_(generator=g)
    out, _ = verify_draft(target, tokens.cuda(), draft, u.cuda(), race.cuda())
    freq = torch.bincount(out[:, 0].cpu().long(), minlength=V) / B
    prob = torch.softmax(p, -1)
    assert bool(((freq - prob).abs() < 6 * torch.sqrt(prob * (1 - prob) / B)).all())


def test_the_residual_may_be_smaller_than_normal_numbers():
    """A refusal whose residual is nothing but probabilities below 2^-126: the draw is among those."""
    V = 3000
    target, draft = torch.full((2, 2, V), -95.0), torch.full((2, 1, V), -math.inf)
    target[:, :, 17], draft[:, :, 17] = 0.0, 0.0
    tokens, u = torch.full((2, 1), 17, dtype=torch.int32), torch.ones((2, 1))
    race = 0.5 + torch.rand((2, V), generator=torch.Generator().manual_seed(9))
    race[0, 2001], race[1, 5] = 1e-3, 1e-3
    check(target, tokens, draft, u, race)
    assert verify_draft(*(t.cuda() for t in (target, tokens, draft, u, race)))[0][:, 0].tolist() == [2001, 5]


def exact_weights(z, n):
    """(rho(z) rho(-max))^n as float32 arithmetic with correctly rounded operations gives it."""
    import numpy as np

    def rho32(x):
        rad = (x.astype(np.float64) ** 2 + 1).astype(np.float32)
        t = np.abs(x) + np.sqrt(rad)
        return np.where(x >= 0, t, np.float32(1) / t)

    z = z.numpy()
    w = rho32(z) * rho32(-z.max(axis=-1, keepdims=True))
    for _ in range(n.bit_length() - 1):
        w = w * w
    assert w.dtype == np.float32
    return torch.from_numpy(w.astype(np.float64))


@pytest.mark.parametrize("n", [8, 32, 64, 256])
def test_close_races_are_decided_exactly(n):
    """Columns whose ratios lie within 1e-5 of each other, the winner 4e-6 above the rest (the sum's rounding and
    those of two divisions are 2e-7): powers above 32 are the C entry's."""
    B, V = 24, 4000
    g = torch.Generator().manual_seed(10 + n)
    half = 0.3 if n <= 64 else 0.1  # no weight below 1e-23
    z = (2 * half * torch.rand((B, V), generator=g) - half).float()
    z[:, ::4] = half  # the row's maximum in every 16 bytes: whichever the kernel refers its weights to is this one
    w = exact_weights(z, n)
    best = torch.randint(0, V, (B,), generator=g)
    gap = 4e-6 + 6e-6 * torch.rand((B, V), generator=g, dtype=torch.float64)
    gap[torch.arange(B), best] = 0.0
    race = (w / w.sum(dim=-1, keepdim=True) * V * (1 + gap)).float()
    # the variates' own rounding, 2^-24, is part of the inputs
    out, accepted = torch.empty((B, 1), dtype=torch.int32, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    zd, rd = z[:, None].contiguous().cuda(), race.cuda()
    torch.cuda.synchronize()
    L.check(L.lib().algx_verify_draft(L.ALGX_HEAD_ALG_CE, n, 1.0, zd.data_ptr(), None, None, None, None, rd.data_ptr(),
                                      out.data_ptr(), accepted.data_ptr(), B, 0, V, L.ALGX_F32, L.stream_of(zd)), "verify")
    assert out[:, 0].tolist() == best.tolist() and accepted.tolist() == [0] * B


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["ce", "alg_ce"])
@pytest.mark.parametrize("B", [1, 40, 64])
def test_sampling_over_a_real_vocabulary(B, kind, dtype):
    target, tokens, _, u, race = inputs(B, 0, 50304, dtype, kind, 2.0, 30 + B)
    check(target, tokens, None, u, race, kind=kind, n=8, c=2.0)
