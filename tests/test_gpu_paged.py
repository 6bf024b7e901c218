"""Paged cache operators against their 64-bit restatement (oracle/serving_math.py)."""

import math

import pytest
import torch

from algx import _lib as L
from algx.kernels.paged import cache_append, cache_evict, paged_attention
from oracle import serving_math as O

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
BAD_PAGE = 8


def make_cache(B, Hkv, page, max_pages, dtype, seed, gain=1.0):
    """CPU pages in shuffled order with spare ones, and the table."""
    g = torch.Generator().manual_seed(seed)
    num = B * max_pages + 3
    k = (gain * torch.randn((num, Hkv, page, 64), generator=g)).to(dtype)
    v = torch.randn((num, Hkv, page, 64), generator=g).to(dtype)
    table = torch.randperm(num, generator=g)[:B * max_pages].reshape(B, max_pages).to(torch.int32)
    return k, v, table, g


def poison(pages, table, lens):
    """NaN wherever no sequence has a cached slot."""
    out = torch.full_like(pages, math.nan)
    size = pages.shape[2]
    for b, n in enumerate(lens):
        for s in range(n):
            p = int(table[b, s // size])
            out[p, :, s % size] = pages[p, :, s % size]
    return out


def bound(mag, ref, dtype, n, kind, top, q, k):
    """Largest error of an output. Scores: 64 products and sums in fp32, each within 2^-24 of
    |q||k| scale (the tensor cores' truncating sums: twice that). Weights: n times the score's
    error plus 2^-21 a factor (root, reciprocal, product), or the exponential's 2^-21 and its
    argument's rounding; the weighted sum errs by twice that relative to sum p|v|. bf16: weights
    rounded to 8 bits (2^-9 of sum p|v|) and the output once (2^-9)."""
    qk = float(q.float().norm(dim=-1).max() * torch.nan_to_num(k.float()).norm(dim=-1).max())
    dx = 2 * 64 * 2.0 ** -24 * qk / 8
    power = n if kind == "asinh" else 1
    dw = 2 * (power * (dx + 2.0 ** -21) + 2.0 ** -22 * top + 2.0 ** -18)
    if dtype == BF16:
        return (dw + 2.0 ** -9) * mag + 2.0 ** -8 * ref.abs() + 1e-30
    return dw * mag + 2.0 ** -23 * ref.abs() + 1e-30


def check_attention(B, T, Hq, Hkv, page, lens, dtype, kind, seed, n=16, c=8.0, window=None, first=0, sink=False,
                    scored=False, gain=1.0, in_place=False, wide=0):
    max_pages = max(1, -(-max(max(lens), 1) // page)) + 1
    k, v, table, g = make_cache(B, Hkv, page, max_pages, dtype, seed, gain)
    k, v = poison(k, table, lens), poison(v, table, lens)
    q = (gain * torch.randn((B, T, Hq, 64), generator=g)).to(dtype)
    s = torch.randn(Hq, generator=g) * c if sink else None
    S = max_pages * page
    scores = torch.rand((B, Hkv, S), generator=g) if scored else None
    ref, new, mag, top = O.paged_attention(q, k, v, table, lens, s, kind=kind, n=n, c=c, window=window, first=first,
                                           scores=scores)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    table = torch.nn.functional.pad(table, (0, wide))  # pages that no sequence has reached
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    sc = dev(scores)
    out = None if not scored or in_place else torch.full_like(sc, math.nan)
    got = paged_attention(dev(q), dev(k), dev(v), dev(table), lens_d, dev(s), kind=kind, n=n, c=c, window=window,
                          first=first, scores=sc, scores_out=out)
    o = got[0] if scored else got
    lim = bound(mag, ref, dtype, n, kind, top, q, k)
    err = (o.double().cpu() - ref).abs()
    assert o.dtype == dtype and bool((err <= lim).all()), float((err / lim).max())
    if scored:
        got_new = got[1]
        assert got_new.data_ptr() == (sc if in_place else out).data_ptr()
        # a slot's sum of at most T Hq / Hkv weights, each within dw of itself, plus the old value's rounding
        dw = float((bound(torch.ones(1), torch.zeros(1), F32, n, kind, top, q, k)).max())
        lim = dw * (new - torch.where(torch.arange(S) < torch.tensor(lens)[:, None, None] - T, scores.double(), 0.0)
                    ).abs() + 2.0 ** -22 * new.abs() + 1e-30
        assert bool(((got_new.double().cpu() - new).abs() <= lim).all())
    assert L.device_error() == 0


CASES = [
    dict(B=1, T=1, Hq=12, Hkv=12, page=64, lens=[300]),
    dict(B=3, T=1, Hq=4, Hkv=4, page=16, lens=[0, 1, 17]),
    dict(B=4, T=1, Hq=2, Hkv=1, page=32, lens=[31, 32, 33, 640], sink=True),
    dict(B=2, T=3, Hq=8, Hkv=2, page=64, lens=[1, 130], sink=True),       # fewer slots than new tokens
    dict(B=2, T=5, Hq=4, Hkv=4, page=16, lens=[5, 260]),
    dict(B=2, T=9, Hq=10, Hkv=2, page=128, lens=[100, 257]),              # 45 rows a head: ragged row tiles
    dict(B=2, T=1, Hq=6, Hkv=3, page=256, lens=[700, 3], window=64, first=4),
    dict(B=2, T=4, Hq=6, Hkv=3, page=16, lens=[333, 40], window=33, first=5, sink=True),
    dict(B=1, T=2, Hq=2, Hkv=2, page=32, lens=[200], window=1, first=0),
    dict(B=1, T=1, Hq=2, Hkv=2, page=32, lens=[200], window=150, first=100),  # the two ranges meet
    dict(B=2, T=1, Hq=4, Hkv=4, page=64, lens=[1500, 90], scored=True, sink=True),
    dict(B=2, T=3, Hq=8, Hkv=4, page=32, lens=[70, 2], scored=True, in_place=True),
    dict(B=1, T=2, Hq=4, Hkv=2, page=16, lens=[500], scored=True, window=100, first=3),
    dict(B=2, T=1, Hq=16, Hkv=2, page=64, lens=[129, 64], scored=True),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["asinh", "softmax"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention(i, kind, dtype):
    check_attention(dtype=dtype, kind=kind, seed=100 + i, **CASES[i])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind,n,gain", [("asinh", 2, 1.0), ("asinh", 32, 6.0), ("asinh", 64, 1.0), ("softmax", 16, 4.0)])
def test_attention_powers_and_score_ranges(kind, n, gain, dtype):
    check_attention(B=2, T=2, Hq=4, Hkv=2, page=32, lens=[260, 47], dtype=dtype, kind=kind, seed=7, n=n, c=2.0,
                    gain=gain, sink=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_widest_window_with_fewer_slots_than_tokens(dtype):
    check_attention(B=2, T=9, Hq=4, Hkv=2, page=16, lens=[3, 40], dtype=dtype, kind="asinh", seed=8, window=2 ** 31 - 1,
                    first=2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sink", [False, True])
def test_attention_of_empty_sequences_alone(dtype, sink):
    for B, T, max_pages in ((1, 1, 1), (3, 2, 200)):
        k, v, table, g = make_cache(B, 2, 16, max_pages, dtype, 14)
        q = torch.randn((B, T, 4, 64), generator=g).to(dtype).cuda()
        lens = torch.zeros(B, dtype=torch.int32).cuda()
        s = torch.ones(4).cuda() if sink else None
        o = paged_attention(q, k.cuda(), v.cuda(), table.cuda(), lens, s, kind="asinh")
        assert bool((o == 0).all())
        scores = torch.ones((B, 2, 16 * max_pages), device="cuda")
        o, new = paged_attention(q, k.cuda(), v.cuda(), table.cuda(), lens, s, scores=scores)
        assert bool((o == 0).all()) and bool((new == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["asinh", "softmax"])
@pytest.mark.parametrize("i", [i for i, case in enumerate(CASES) if not case.get("scored")])
def test_attention_with_wide_tables(i, kind, dtype):
    """Short tables are joined by clusters, wide ones along the line of all groups."""
    check_attention(dtype=dtype, kind=kind, seed=100 + i, wide=4096, **CASES[i])


def test_attention_long_cache_of_many_splits():
    check_attention(B=1, T=1, Hq=2, Hkv=1, page=64, lens=[9001], dtype=BF16, kind="asinh", seed=3, scored=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,lens,sink", [(1, 1, [40007], False), (2, 3, [9001, 0], True)])
def test_attention_few_rows_of_many_parts(B, T, lens, sink, dtype):
    """A few rows of hundreds of partial results, and of none."""
    check_attention(B=B, T=T, Hq=2, Hkv=1, page=128, lens=lens, dtype=dtype, kind="asinh", seed=4, sink=sink)


def test_attention_rows_see_nothing_of_later_tokens():
    """Infinities and NaN in the newest token's key and value stay out of the earlier tokens' outputs."""
    B, T, H, page = 1, 3, 2, 16
    for value in (math.inf, math.nan):
        for dtype in (BF16, F32):
            k, v, table, g = make_cache(B, H, page, 3, dtype, 5)
            q = torch.randn((B, T, H, 64), generator=g).to(dtype).cuda()
            lens = torch.tensor([37], dtype=torch.int32).cuda()
            want = paged_attention(q, k.cuda(), v.cuda(), table.cuda(), lens, kind="asinh", c=8.0)
            k[int(table[0, 36 // page]), :, 36 % page] = value
            v[int(table[0, 36 // page]), :, 36 % page] = value
            got = paged_attention(q, k.cuda(), v.cuda(), table.cuda(), lens, kind="asinh", c=8.0)
            assert torch.equal(got[:, :2], want[:, :2])
            assert not bool(torch.isfinite(got[:, 2]).all())


def test_attention_strided_queries_and_another_stream():
    k, v, table, g = make_cache(2, 2, 32, 4, BF16, 9)
    q = torch.randn((2, 4, 3, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([100, 50], dtype=torch.int32).cuda()
    k, v, table = k.cuda(), v.cuda(), table.cuda()
    want = paged_attention(q.transpose(1, 2).contiguous(), k, v, table, lens)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = paged_attention(q.transpose(1, 2), k, v, table, lens)
    st.synchronize()
    assert torch.equal(got, want)


def test_attention_repeats_bit_for_bit_and_in_a_graph():
    k, v, table, g = make_cache(2, 4, 64, 8, BF16, 10)
    q = torch.randn((2, 1, 8, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([500, 130], dtype=torch.int32).cuda()
    k, v, table = k.cuda(), v.cuda(), table.cuda()
    run = lambda: paged_attention(q, k, v, table, lens, kind="asinh", c=8.0)  # noqa: E731
    want = run()
    assert torch.equal(run(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    lens.fill_(200)
    graph.replay()
    assert torch.equal(got, run()) and not torch.equal(got, want)


def test_attention_pages_beyond_32_bit_offsets():
    """Pages whose element offsets pass 2^31 and whose byte offsets pass 2^32."""
    page, H = 256, 8
    num = 2 ** 31 // (page * H * 64) + 40
    k, v = (torch.empty((num, H, page, 64), dtype=BF16, device="cuda") for _ in range(2))
    small_k, small_v, _, g = make_cache(1, H, page, 4, BF16, 11)
    high = torch.tensor([num - 1, 0, num - 30, num - 2], device="cuda")
    k[high], v[high] = small_k[:4].cuda(), small_v[:4].cuda()
    q = torch.randn((1, 1, H, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([1000], dtype=torch.int32).cuda()
    low = torch.arange(4, dtype=torch.int32)[None].cuda()
    want = paged_attention(q, small_k.cuda(), small_v.cuda(), low, lens)
    assert torch.equal(paged_attention(q, k, v, high.to(torch.int32)[None], lens), want)
    qkv = torch.randn((1, 3, 3 * H, 64), generator=g).to(BF16).cuda()
    cache_append(qkv, k, v, high.to(torch.int32)[None], lens)
    assert torch.equal(v[num - 2, :, 1000 - 768:1003 - 768], qkv[0, :, 2 * H:].transpose(0, 1))


def test_attention_skips_what_the_table_gets_wrong():
    k, v, table, g = make_cache(2, 2, 16, 4, BF16, 12)
    q = torch.randn((2, 1, 2, 64), generator=g).to(BF16).cuda()
    k, v = k.cuda(), v.cuda()
    bad = table.clone()
    bad[0, 1], bad[1, 2] = -5, 10 ** 6
    lens = torch.tensor([60, 10 ** 9], dtype=torch.int32).cuda()
    o = paged_attention(q, k, v, bad.cuda(), lens)
    assert bool(torch.isfinite(o.float()).all()) and L.device_error() & BAD_PAGE
    lens = torch.tensor([-3, 5], dtype=torch.int32).cuda()
    o = paged_attention(q, k, v, table.cuda(), lens)
    assert bool((o[0] == 0).all()) and bool((o[1] != 0).any()) and L.device_error() == 0


def test_attention_of_no_sequences_or_no_tokens():
    k, v, table, _ = make_cache(1, 2, 16, 2, BF16, 13)
    k, v = k.cuda(), v.cuda()
    none = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    o = paged_attention(torch.empty((0, 1, 2, 64), dtype=BF16, device="cuda"), k, v, none, none[:, 0])
    assert o.shape == (0, 1, 2, 64)
    lens = torch.tensor([4], dtype=torch.int32).cuda()
    o = paged_attention(torch.empty((1, 0, 2, 64), dtype=BF16, device="cuda"), k, v, table.cuda(), lens)
    assert o.shape == (1, 0, 2, 64)


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("norm,rot", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("B,T,Hq,Hkv,page,lens,counts,positions", [
    (1, 1, 12, 12, 64, [0], None, None),
    (3, 1, 6, 2, 16, [15, 16, 31], None, [40, 2, 7]),
    (2, 37, 5, 1, 16, [10, 0], [37, 4], None),
    (2, 130, 12, 12, 64, [3, 60], None, None),
    (1, 3, 1, 3, 32, [61], [0], None),
])
def test_append(B, T, Hq, Hkv, page, lens, counts, positions, norm, rot, dtype):
    max_pages = -(-(max(lens) + T) // page)
    k, v, table, g = make_cache(B, Hkv, page, max_pages, dtype, 20 + T)
    qkv = torch.randn((B, T, Hq + 2 * Hkv, 64), generator=g).to(dtype)
    gq, gk = (1 + 0.3 * torch.randn(64, generator=g) for _ in range(2))
    ang = torch.rand((max_pages * page + 64, 32), generator=g) * 6
    opts = dict(rotary=(torch.cos(ang), torch.sin(ang)) if rot else None)
    gains = (gq, gk) if norm else (None, None)
    ref_q, ref_k, ref_v = O.cache_append(qkv, k, v, table, lens, *gains, positions=positions, counts=counts, **opts)
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    kd, vd = k.cuda(), v.cuda()
    where = torch.full((B, Hkv, max_pages * page), -7, dtype=torch.int32, device="cuda")
    q = cache_append(qkv.cuda(), kd, vd, table.cuda(), i32(lens), *(None if x is None else x.cuda() for x in gains),
                     rotary=None if not rot else tuple(x.cuda() for x in opts["rotary"]), positions=i32(positions),
                     counts=i32(counts), slot_positions=where)
    # fp32 evaluation: 64 squares in the norm, five products and one sum after it, each 2^-24 of
    # at most |y| (rotation: of both halves); then one rounding to bf16 (2^-9)
    eps = 2.0 ** -20 if norm or rot else 0.0
    for got, ref in ((q, ref_q), (kd, ref_k)):
        got, half = got.double().cpu(), ref.abs() + ref.abs().roll(32, -1)
        lim = eps * half + (2.0 ** -8 * ref.abs() if dtype == BF16 else 0) + 1e-30
        assert bool(((got - ref).abs() <= lim).all())
    assert torch.equal(vd.double().cpu(), ref_v)
    for b in range(B):
        n = T if counts is None else counts[b]
        want = torch.full((max_pages * page,), -7, dtype=torch.int32)
        start = lens[b] if positions is None else positions[b]
        want[lens[b]:lens[b] + n] = torch.arange(start, start + n, dtype=torch.int32)
        assert torch.equal(where[b].cpu(), want.expand(Hkv, -1))
    assert L.device_error() == 0


def test_append_keeps_out_of_what_does_not_fit():
    k, v, table, g = make_cache(2, 2, 16, 2, BF16, 30)
    kd, vd = k.cuda(), v.cuda()
    table[1, 1] = 10 ** 6
    qkv = torch.randn((2, 4, 6, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([30, 14], dtype=torch.int32).cuda()
    cache_append(qkv, kd, vd, table.cuda(), lens)  # slots 32, 33 and a page that does not exist
    assert L.device_error() & BAD_PAGE
    changed = (vd.cpu() != v).any(dim=-1).any(dim=1).nonzero().tolist()
    assert sorted(changed) == sorted([[int(table[0, 1]), 14], [int(table[0, 1]), 15],
                                      [int(table[1, 0]), 14], [int(table[1, 0]), 15]])


def test_append_position_outside_the_tables_is_flagged():
    k, v, table, g = make_cache(1, 1, 16, 2, BF16, 31)
    rot = tuple(torch.rand((8, 32), generator=g).cuda() for _ in range(2))
    qkv = torch.randn((1, 2, 3, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([7], dtype=torch.int32).cuda()
    q = cache_append(qkv, k.cuda(), v.cuda(), table.cuda(), lens, rotary=rot)
    assert bool(torch.isfinite(q.float()).all()) and L.device_error() & BAD_PAGE


# ------------------------------------------------------------------- eviction
def check_evict(B, Hkv, page, lens, budget, first, recent, dtype, seed, scores=None, levels=0):
    max_pages = max(1, -(-max(lens) // page))
    S = max_pages * page
    k, v, table, g = make_cache(B, Hkv, page, max_pages, dtype, seed)
    if scores is None:
        scores = torch.rand((B, Hkv, S), generator=g)
        if levels:  # many equal scores
            scores = torch.floor(scores * levels)
    positions = torch.stack([torch.stack([torch.cat([torch.randperm(n, generator=g), torch.full((S - n,), 99999)])
                                          for _ in range(Hkv)]) for n in lens]).to(torch.int32)
    args = [t.cuda() for t in (k, v, table, torch.tensor(lens, dtype=torch.int32), scores, positions)]
    new_lens, new_scores, new_positions, kept = cache_evict(*args, budget=budget, first=first, recent=recent)
    assert torch.equal(args[4].cpu().nan_to_num(nan=-1), scores.nan_to_num(nan=-1))
    assert torch.equal(args[3].cpu(), torch.tensor(lens, dtype=torch.int32))
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    kk, vv = k.clone(), v.clone()
    for b, n in enumerate(lens):
        for h in range(Hkv):
            plan = O.evict_plan(scores[b, h], positions[b, h], n, budget, first, recent)
            assert kept[b, h].tolist() == plan + [-1] * (budget - len(plan))
            assert torch.equal(new_scores[b, h, :len(plan)].cpu().nan_to_num(nan=-1),
                               scores[b, h, plan].nan_to_num(nan=-1))
            assert torch.equal(new_positions[b, h, :len(plan)].cpu(), positions[b, h, plan])
            assert bool((new_scores[b, h, len(plan):] == 0).all()) and bool((new_positions[b, h, len(plan):] == -1).all())
            for to, of in enumerate(plan):
                if to != of:
                    at, src = (int(table[b, to // page]), h, to % page), (int(table[b, of // page]), h, of % page)
                    kk[at], vv[at] = k[src], v[src]
    assert torch.equal(args[0].cpu(), kk) and torch.equal(args[1].cpu(), vv)
    again = cache_evict(*args, budget=budget, first=first, recent=recent)
    for x, y in zip(again, (new_lens, new_scores, new_positions, kept)):
        assert torch.equal(x.nan_to_num(nan=-1) if x.is_floating_point() else x,
                           y.nan_to_num(nan=-1) if y.is_floating_point() else y)
    assert torch.equal(args[0].cpu(), kk) and L.device_error() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Hkv,page,lens,budget,first,recent,levels", [
    (1, 1, 16, [40], 20, 2, 5, 0),
    (3, 2, 16, [0, 1, 33], 1, 0, 1, 0),
    (2, 3, 64, [700, 699], 300, 4, 50, 7),
    (2, 2, 32, [64, 2100], 64, 0, 0, 0),
    (2, 2, 32, [2000, 1999], 1998, 4, 1000, 3),
    (1, 2, 128, [5000], 1025, 4, 1021, 0),   # nothing but the protected slots
    (2, 1, 16, [30, 31], 500, 4, 8, 0),      # under budget
    (1, 1, 256, [1025], 1024, 0, 0, 1),      # every score equal
])
def test_evict(B, Hkv, page, lens, budget, first, recent, levels, dtype):
    check_evict(B, Hkv, page, lens, budget, first, recent, dtype, 40 + budget, levels=levels)


def test_evict_of_more_slots_than_shared_memory_holds():
    check_evict(1, 1, 256, [51000], 3000, 4, 100, BF16, 60)


def test_evict_odd_scores():
    """Negative, infinite, NaN and signed-zero scores rank as documented."""
    pool = torch.tensor([-1.0, 0.0, -0.0, math.inf, -math.inf, math.nan, 3.0, 1e-40])
    g = torch.Generator().manual_seed(1)
    scores = pool[torch.randint(0, 8, (2, 2, 128), generator=g)]
    check_evict(2, 2, 16, [128, 77], 50, 1, 3, BF16, 50, scores=scores)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_evict_keeps_protected_slots_above_infinite_scores(dtype):
    """Infinite scores in the low slots, more of them than the budget has room for beside the protected positions."""
    scores = torch.rand((2, 2, 160), generator=torch.Generator().manual_seed(2))
    scores[:, :, :100] = math.inf
    check_evict(2, 2, 16, [160, 131], 40, 5, 20, dtype, 51, scores=scores)


def test_evict_of_no_sequences():
    k, v, _, _ = make_cache(1, 2, 16, 2, BF16, 13)
    table = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    out = cache_evict(k.cuda(), v.cuda(), table, table[:, 0], torch.empty((0, 2, 32), device="cuda"),
                      torch.empty((0, 2, 32), dtype=torch.int32, device="cuda"), budget=4)
    assert [tuple(t.shape) for t in out] == [(0,), (0, 2, 32), (0, 2, 32), (0, 2, 4)]


def test_operators_match_the_functions():
    from algx import torch_ops as T
    k, v, table, g = make_cache(2, 2, 32, 4, BF16, 70)
    qkv = torch.randn((2, 3, 8, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([60, 5], dtype=torch.int32).cuda()
    gains = [torch.rand(64, generator=g).cuda() for _ in range(2)]
    table = table.cuda()
    caches = [(k.cuda(), v.cuda()) for _ in range(2)]
    qs = [f(qkv, *c, table, lens, *gains) for f, c in zip((cache_append, T.cache_append), caches)]
    assert torch.equal(*qs) and all(torch.equal(a, b) for a, b in zip(*caches))
    after = lens + 3
    scores = [torch.rand((2, 2, 128), generator=torch.Generator().manual_seed(1)).cuda() for _ in range(2)]
    a = paged_attention(qs[0], *caches[0], table, after, kind="asinh", c=8.0, scores=scores[0])
    b = T.paged_attention(qs[0], *caches[1], table, after, kind="asinh", c=8.0, scores=scores[1])
    assert torch.equal(a[0], b[0]) and torch.equal(scores[0], scores[1])
    assert torch.equal(paged_attention(qs[0], *caches[0], table, after, window=9),
                       T.paged_attention(qs[0], *caches[0], table, after, window=9))
    pos = torch.arange(128, dtype=torch.int32).expand(2, 2, 128).contiguous().cuda()
    outs = [f(*c, table, after, scores[0], pos, budget=20, recent=4) for f, c in
            zip((cache_evict, T.cache_evict), caches)]
    assert all(torch.equal(x, y) for x, y in zip(*outs)) and all(torch.equal(x, y) for x, y in zip(*caches))


def test_the_attention_operator_takes_what_the_function_takes():
    """A number for the sink, and scores into a buffer of their own."""
    from algx import torch_ops as T
    k, v, table, g = make_cache(2, 2, 32, 4, BF16, 72)
    k, v, table = k.cuda(), v.cuda(), table.cuda()
    q = torch.randn((2, 3, 4, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([60, 5], dtype=torch.int32).cuda()
    assert torch.equal(T.paged_attention(q, k, v, table, lens, 1.5, kind="asinh", c=8.0),
                       paged_attention(q, k, v, table, lens, 1.5, kind="asinh", c=8.0))
    scores = torch.rand((2, 2, 128), generator=g).cuda()
    before, out = scores.clone(), [torch.full_like(scores, math.nan) for _ in range(2)]
    a = paged_attention(q, k, v, table, lens, 0.5, scores=scores, scores_out=out[0])
    b = T.paged_attention(q, k, v, table, lens, 0.5, scores=scores, scores_out=out[1])
    assert torch.equal(a[0], b[0]) and b[1] is out[1] and torch.equal(*out) and torch.equal(scores, before)
    c = T.paged_attention(q, k, v, table, lens, 0.5, scores=scores, scores_out=scores)
    assert torch.equal(c[0], a[0]) and torch.equal(scores, out[0])


def test_unaligned_inputs_are_copied():
    k, v, table, g = make_cache(1, 2, 16, 2, BF16, 71)
    base = torch.randn(1 + 6 * 64, generator=g).to(BF16).cuda()
    qkv = base[1:].view(1, 1, 6, 64)
    gains = torch.rand(130, generator=g).cuda()
    lens = torch.tensor([3], dtype=torch.int32).cuda()
    caches = [(k.cuda(), v.cuda()) for _ in range(2)]
    a = cache_append(qkv, *caches[0], table.cuda(), lens, gains[1:65], gains[65:129])
    b = cache_append(qkv.clone(), *caches[1], table.cuda(), lens, gains[1:65].clone(), gains[65:129].clone())
    assert torch.equal(a, b) and torch.equal(caches[0][0], caches[1][0])
    odd = torch.empty(1 + a.numel(), dtype=BF16, device="cuda")[1:].view(a.shape)
    odd.copy_(a)
    assert torch.equal(paged_attention(odd, *caches[0], table.cuda(), lens + 1),
                       paged_attention(a, *caches[0], table.cuda(), lens + 1))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("in_place", [False, True])
def test_scores_of_a_call_without_tokens(in_place, dtype):
    """The cached slots' scores as they were, zeros beyond them."""
    k, v, table, g = make_cache(3, 2, 16, 70, dtype, 15)
    S = 70 * 16
    scores = torch.rand((3, 2, S), generator=g)
    lens = [0, 1, 777]
    want = torch.where(torch.arange(S) < torch.tensor(lens)[:, None, None], scores, 0.0)
    sc = scores.cuda()
    out = sc if in_place else torch.full_like(sc, math.nan)
    q = torch.empty((3, 0, 4, 64), dtype=dtype, device="cuda")
    o, got = paged_attention(q, k.cuda(), v.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                             scores=sc, scores_out=out)
    assert o.shape == (3, 0, 4, 64) and got.data_ptr() == out.data_ptr()
    assert torch.equal(got.cpu(), want) and L.device_error() == 0


def test_other_threads_run_while_a_launch_waits():
    """The stream's queue is full behind a kernel of some 0.4 s: a thread that looks at the clock every millisecond is
    not held up as long as the calls are."""
    import threading
    import time
    k, v, table, g = make_cache(1, 2, 16, 4, BF16, 73)
    k, v, table = k.cuda(), v.cuda(), table.cuda()
    qkv = torch.randn((1, 1, 6, 64), generator=g).to(BF16).cuda()
    lens = torch.tensor([5], dtype=torch.int32).cuda()
    calls = [lambda: cache_append(qkv, k, v, table, lens), lambda: paged_attention(qkv[:, :, :4], k, v, table, lens)]
    for call in calls:
        call()
        torch.cuda.synchronize()
        ticks, stop = [], threading.Event()

        def tick():
            while not stop.is_set():
                ticks.append(time.perf_counter())
                time.sleep(1e-3)

        thread = threading.Thread(target=tick)
        thread.start()
        torch.cuda._sleep(800_000_000)
        worst = 0.0
        for _ in range(3000):
            t0 = time.perf_counter()
            call()
            worst = max(worst, time.perf_counter() - t0)
        stop.set()
        thread.join()
        torch.cuda.synchronize()
        gap = max(b - a for a, b in zip(ticks, ticks[1:]))
        assert worst > 0.1, "no call waited: the queue was never full"
        assert gap < 0.5 * worst


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["asinh", "softmax"])
@pytest.mark.parametrize("case", [
    dict(B=2, T=70, Hq=3, Hkv=3, page=16, lens=[200, 75], sink=True),                     # a chunk of a prompt
    dict(B=2, T=64, Hq=2, Hkv=2, page=64, lens=[64, 131], scored=True, in_place=True),
    dict(B=1, T=33, Hq=6, Hkv=2, page=32, lens=[300], window=40, first=3),                # 99 rows a head
    dict(B=3, T=40, Hq=4, Hkv=2, page=128, lens=[20, 0, 170], scored=True, sink=True),    # fewer slots than tokens
    dict(B=1, T=17, Hq=2, Hkv=2, page=16, lens=[260], scored=True, window=30, first=2),
])
def test_attention_of_prompt_chunks(case, kind, dtype):
    """More rows than three tiles hold, in both joins."""
    check_attention(dtype=dtype, kind=kind, seed=300 + case["T"], **case)
    if not case.get("scored"):
        check_attention(dtype=dtype, kind=kind, seed=300 + case["T"], wide=4096, **case)
