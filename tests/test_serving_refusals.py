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
                 new_scores=base + 2048, new_positions=base + 3072, kept=base + 4096, workspace=base)
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
