"""Host side of serving: the page accounting of the cache (CPU only)."""

import pytest
import torch

from algx.serve import PagedCache, head_options


def cache(**kw):
    return PagedCache(2, 3, 4, 100, page_size=16, device="cpu", **kw)


def test_pages_are_handed_out_once_and_come_back():
    c = cache()
    assert c.slots == 112 and len(c.free) == 28 and c.k.shape == (2, 28, 3, 16, 64)
    c.reserve([1, 16, 17, 100])
    assert [len(o) for o in c.owned] == [1, 1, 2, 7]
    pages = [p for o in c.owned for p in o]
    assert len(set(pages)) == len(pages) == 28 - len(c.free)
    for b, own in enumerate(c.owned):
        assert c.table[b, :len(own)].tolist() == own
    before = [list(o) for o in c.owned]
    c.reserve([1, 16, 17, 100])          # nothing more is needed
    c.reserve([0, 0, 0, 0])              # and nothing is taken away
    assert c.owned == before
    c.trim([1, 0, 16, 33])
    assert [len(o) for o in c.owned] == [1, 0, 1, 3] and len(c.free) == 28 - 5
    c.release(3)
    assert c.owned[3] == [] and len(c.free) == 26
    c.reserve([112, 112, 0, 0])
    assert len({p for o in c.owned for p in o}) == 15


def test_running_out_of_pages_changes_nothing():
    c = cache(pages=5)
    c.reserve([16, 16, 0, 0])
    table, owned = c.table.clone(), [list(o) for o in c.owned]
    with pytest.raises(MemoryError):
        c.reserve([48, 48, 16, 16])
    assert torch.equal(c.table, table) and c.owned == owned and len(c.free) == 3


def test_bounds():
    c = cache()
    with pytest.raises(ValueError, match="at most 112 slots"):
        c.reserve([113, 0, 0, 0])
    with pytest.raises(ValueError, match="at most 112 slots"):
        c.reserve([1, 1])
    with pytest.raises(ValueError, match="must be positive"):
        PagedCache(1, 1, 0, 16, device="cpu")


def test_head_options_follow_the_model():
    from algx.model import config_125m, config_algebraic_125m
    assert head_options(config_125m(), 0.5) == dict(kind="ce", temperature=0.5)
    assert head_options(config_algebraic_125m()) == dict(kind="alg_ce", n=8, c=2.0)


def test_operators_have_shapes_for_tracers():
    """The serving operators' fake implementations give the shapes and dtypes of the real ones."""
    from algx import torch_ops as T
    from torch._subclasses.fake_tensor import FakeTensorMode
    bf16, i32 = torch.bfloat16, torch.int32
    with FakeTensorMode():
        k = torch.empty((9, 2, 16, 64), dtype=bf16)
        v, table, lens = torch.empty_like(k), torch.empty((3, 4), dtype=i32), torch.empty(3, dtype=i32)
        q = T.cache_append(torch.empty((3, 5, 8, 64), dtype=bf16), k, v, table, lens)
        assert q.shape == (3, 5, 4, 64) and q.dtype == bf16
        assert T.paged_attention(q, k, v, table, lens, kind="asinh").shape == q.shape
        scores, pos = torch.empty((3, 2, 64)), torch.empty((3, 2, 64), dtype=i32)
        o, s = T.paged_attention(q, k, v, table, lens, scores=scores)
        assert o.shape == q.shape and s is scores
        out = T.cache_evict(k, v, table, lens, scores, pos, budget=7)
        assert [tuple(t.shape) for t in out] == [(3,), (3, 2, 64), (3, 2, 64), (3, 2, 7)]
        assert [t.dtype for t in out] == [i32, torch.float32, i32, i32]
        tokens, accepted = T.verify_draft(torch.empty((3, 5, 99)), torch.empty((3, 4), dtype=i32), None,
                                          torch.empty((3, 4)), torch.empty((3, 99)))
        assert tokens.shape == (3, 5) and accepted.shape == (3,) and tokens.dtype == accepted.dtype == i32
    with pytest.raises(ValueError, match="window must be positive"):
        T.paged_attention(None, None, None, None, None, window=0)


def test_the_algebraic_head_has_no_temperature():
    """As ``verify_draft`` refuses it: a temperature that is ignored would sample from another distribution than asked."""
    from algx.model import config_algebraic_125m
    with pytest.raises(ValueError, match="temperature is for the ce kind"):
        head_options(config_algebraic_125m(), 0.5)


def test_the_attention_operator_has_the_functions_arguments():
    import inspect

    from algx import torch_ops as T
    from algx.kernels import paged
    from torch._subclasses.fake_tensor import FakeTensorMode
    assert inspect.signature(T.paged_attention) == inspect.signature(paged.paged_attention)
    with FakeTensorMode():
        k, table = torch.empty((9, 2, 16, 64)), torch.empty((3, 4), dtype=torch.int32)
        args = torch.empty((3, 5, 4, 64)), k, k, table, table[:, 0]
        assert T.paged_attention(*args, 0.5).shape == (3, 5, 4, 64)
        scores, out = torch.empty((3, 2, 64)), torch.empty((3, 2, 64))
        assert T.paged_attention(*args, scores=scores, scores_out=out)[1] is out
    with pytest.raises(ValueError, match="scores_out without scores"):
        T.paged_attention(None, None, None, None, None, scores_out=out)
