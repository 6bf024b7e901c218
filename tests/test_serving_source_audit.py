"""Source audit of the serving kernels: the algebraic kinds compute no exponential or logarithm.

Every exp call in the serving sources stands behind the softmax kind's compile-time
guard, and the cache's kernels have none.
"""

import os

import pytest

from tests.test_source_audit import CSRC, _calls, _code_lines


def test_cache_kernels_have_no_transcendental():
    assert os.path.exists(os.path.join(CSRC, "cache.cu"))
    assert _calls("cache.cu") == []


@pytest.mark.parametrize("name", ["paged_common.cuh", "paged_attn.cu", "verify.cu"])
def test_transcendentals_serve_the_softmax_kind(name):
    lines = _code_lines(name)
    for n, line in _calls(name):
        window = "\n".join(lines[max(0, n - 6):n])
        assert "kSoftmax" in window, f"{name}:{n}: {line.strip()}"


def test_the_softmax_kind_does_use_them():
    assert _calls("paged_common.cuh") and _calls("verify.cu")
