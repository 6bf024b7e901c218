"""The serving entries of the C ABI refuse what their kernels could not address (CPU only: every call is refused by
its arguments alone, before anything is launched)."""

import ctypes

import pytest

from algx import _lib as L


def evict(B=1, Hkv=1, page_size=16, max_pages=4, budget=8, dtype=L.ALGX_BF16, **at):
    """Status and message of an eviction whose arrays all stand at one aligned host address unless ``at`` says else."""
    lib = L.lib()
    room = (ctypes.c_char * 8192)()
    base = (ctypes.addressof(room) + 63) // 64 * 64
    place = dict(k=base, v=base, table=base, lens=base, scores=base, positions=base, new_lens=base + 1024,
                 new_scores=base + 2048, new_positions=base + 4096, kept=base + 5120, workspace=base)
    place.update({name: place[name] + off for name, off in at.items()})
    p = place
    # a workspace of one byte is too small: whatever passes the other checks is refused for that
    status = lib.algx_cache_evict(p["k"], p["v"], p["table"], p["lens"], p["scores"], p["positions"], budget, 0, 0,
                                  p["new_lens"], p["new_scores"], p["new_positions"], p["kept"], B, Hkv, 4, page_size,
                                  max_pages, 64, dtype, p["workspace"], 1, None)
    return status, lib.algx_last_error().decode()


def test_evict_reaches_the_last_check():
    status, message = evict()
    assert status == L.ALGX_ERR_INVALID and "workspace too small" in message


@pytest.mark.parametrize("name", ["scores", "positions", "new_scores", "new_positions"])
@pytest.mark.parametrize("off", [4, 8])
def test_evict_needs_aligned_scores_and_positions(name, off):
    """They are read and written four elements at a time."""
    status, message = evict(**{name: off})
    assert status == L.ALGX_ERR_INVALID and "16-byte aligned" in message


@pytest.mark.parametrize("page_size,max_pages,budget,dtype", [
    (256, 2 ** 20, 2 ** 31 - 513, L.ALGX_BF16),
    (256, 2 ** 23 - 9, 2 ** 28 - 257, L.ALGX_BF16),
    (256, 2 ** 23 - 9, 2 ** 27 - 129, L.ALGX_F32),
])
def test_evict_counts_in_32_bits(page_size, max_pages, budget, dtype):
    """The largest tables and budgets whose slots and pieces of moved rows the kernels' 32-bit counters hold, and one
    more (below it a budget leaves rows to move, which bound it earlier)."""
    sizes = dict(page_size=page_size, max_pages=max_pages, dtype=dtype)
    assert "workspace too small" in evict(budget=budget, **sizes)[1]
    status, message = evict(budget=budget + 1, **sizes)
    assert status == L.ALGX_ERR_INVALID and "too large" in message


def test_evict_of_tables_near_32_bits():
    assert "workspace too small" in evict(page_size=16, max_pages=(2 ** 31 - 2049) // 16, budget=8)[1]
    assert "too large" in evict(page_size=16, max_pages=(2 ** 31 - 2049) // 16 + 1, budget=8)[1]


def test_attention_counts_groups_of_slots_in_32_bits():
    """A sequence's last group of 32 slots ends below 2^31."""
    lib = L.lib()
    cfg = L.PagedConfig(0, 16, 0, 0, 1.0, 1.0)
    call = lambda pages: lib.algx_paged_attn(cfg, *[None] * 9, 0, 1, 2, 2, 1, 16, pages, 64, L.ALGX_BF16, None, 0,  # noqa: E731
                                             None)
    assert call(2 ** 27 - 5) == L.ALGX_OK
    for pages in (2 ** 27 - 4, 2 ** 27 - 1, 2 ** 60):
        assert call(pages) == L.ALGX_ERR_INVALID and b"too large" in lib.algx_last_error()


@pytest.mark.parametrize("scale,inv_unit", [(0.0, 1.0), (-1.0, 1.0), (float("inf"), 1.0), (float("nan"), 1.0),
                                            (1.0, float("inf")), (1.0, 0.0)])
def test_attention_needs_a_positive_finite_scale(scale, inv_unit):
    """The largest score of a group is looked for before scaling, and masked scores are -inf times the scale."""
    lib = L.lib()
    cfg = L.PagedConfig(0, 16, 0, 0, scale, inv_unit)
    status = lib.algx_paged_attn(cfg, *[None] * 9, 0, 1, 2, 2, 1, 16, 1, 64, L.ALGX_BF16, None, 0, None)
    assert status == L.ALGX_ERR_INVALID and b"positive and finite" in lib.algx_last_error()


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -1.0, 0.0])
def test_verification_needs_a_positive_finite_scale(scale):
    lib = L.lib()
    status = lib.algx_verify_draft(L.ALGX_HEAD_CE, 2, scale, *[None] * 8, 0, 1, 9, L.ALGX_F32, None)
    assert status == L.ALGX_ERR_INVALID and b"positive and finite" in lib.algx_last_error()


def test_options_whose_reciprocal_float32_does_not_hold():
    """1e-39 is positive and finite, 1e39 is not a float32: the logits' differences of zero times it are NaN."""
    import torch

    from algx.kernels.paged import paged_attention
    from algx.kernels.verify import verify_draft
    none = torch.zeros(1)
    with pytest.raises(ValueError, match="temperature must be"):
        verify_draft(none, none, None, none, none, temperature=1e-39)
    with pytest.raises(ValueError, match="positive and finite"):
        verify_draft(none, none, None, none, none, kind="alg_ce", n=8, c=1e-39)
    with pytest.raises(ValueError, match="positive and finite"):
        paged_attention(none, none, none, none, none, kind="asinh", c=1e-39)
    with pytest.raises(ValueError, match="temperature must be"):  # its reciprocal is zero
        verify_draft(none, none, None, none, none, temperature=1e60)
