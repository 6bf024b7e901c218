"""The serving operators refuse bad arguments before any launch (CPU only)."""

import pytest
import torch

from algx import _lib as L
from algx._lib import AlgxError
from algx.kernels.paged import cache_append, cache_evict, paged_attention
from algx.kernels.verify import verify_draft

BF16, I32 = torch.bfloat16, torch.int32


def cache(heads=2, size=16, D=64, dtype=BF16):
    k = torch.zeros((3, heads, size, D), dtype=dtype)
    return k, k.clone(), torch.zeros((2, 4), dtype=I32), torch.zeros(2, dtype=I32)


def refuses(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


@pytest.mark.parametrize("match,change", [
    ("head_dim 64", dict(D=32)), ("power of two", dict(size=24)), ("power of two", dict(size=8)),
    ("power of two", dict(size=512)), ("bfloat16 or float32", dict(dtype=torch.float16)),
])
def test_cache_layout(match, change):
    k, v, table, lens = cache(**change)
    q = torch.zeros((2, 1, 2, 64), dtype=k.dtype)
    refuses(match, paged_attention, q, k, v, table, lens)
    refuses(match, cache_append, torch.zeros((2, 1, 6, 64), dtype=k.dtype), k, v, table, lens)


def test_cache_shapes():
    k, v, table, lens = cache()
    q = torch.zeros((2, 1, 2, 64), dtype=BF16)
    refuses("one dtype", paged_attention, q, k, v.float(), table, lens)
    refuses("must both have shape", paged_attention, q, k, v[:2], table, lens)
    refuses("contiguous", paged_attention, q, k.transpose(1, 2).contiguous().transpose(1, 2), v, table, lens)
    refuses(r"lens \(B,\)", paged_attention, q, k, v, table, lens[:1])
    refuses("int32", paged_attention, q, k, v, table.long(), lens)


def test_attention_arguments():
    k, v, table, lens = cache()
    q = torch.zeros((2, 1, 2, 64), dtype=BF16)
    call = lambda q=q, **kw: paged_attention(q, k, v, table, lens, **kw)  # noqa: E731
    refuses("multiple of 2", call, q=torch.zeros((2, 1, 3, 64), dtype=BF16))
    refuses("share one dtype", call, q=q.float())
    refuses("unknown attention kernel", call, kind="relu")
    refuses("power of two", call, kind="asinh", n=12)
    refuses("positive and finite", call, kind="asinh", c=0.0)
    refuses("window must be positive", call, window=0)
    refuses("first must not be negative", call, window=4, first=-1)
    refuses("scores must be", call, scores=torch.zeros((2, 2, 63)))
    refuses("scores_out must be", call, scores=torch.zeros((2, 2, 64)), scores_out=torch.zeros((2, 2, 64), dtype=BF16))
    refuses("scores_out without scores", call, scores_out=torch.zeros((2, 2, 64)))
    with pytest.raises(AlgxError, match="CUDA tensors only"):
        call()


def test_append_arguments():
    k, v, table, lens = cache()
    qkv, g = torch.zeros((2, 3, 6, 64), dtype=BF16), torch.ones(64)
    call = lambda qkv=qkv, *a, **kw: cache_append(qkv, k, v, table, lens, *a, **kw)  # noqa: E731
    refuses("qkv must have shape", call, qkv[..., :32])
    refuses("qkv must have shape", call, qkv[:, :, :3])
    refuses("share one dtype", call, qkv.float())
    refuses("both gain_q and gain_k", call, qkv, g)
    refuses("gains must be float32", call, qkv, g, g.to(BF16))
    refuses("eps must be positive", call, qkv, g, g, eps=0.0)
    refuses("rotary tables", call, rotary=(torch.ones((4, 16)), torch.ones((4, 16))))
    refuses("rotary tables", call, rotary=(torch.ones((4, 32)), torch.ones((5, 32))))
    refuses("positions must be int32", call, positions=torch.zeros(2))
    refuses("counts must be int32", call, counts=torch.zeros(3, dtype=I32))
    refuses("slot_positions must be", call, slot_positions=torch.zeros((2, 2, 64)))
    with pytest.raises(AlgxError, match="CUDA tensors only"):
        call()


def test_evict_arguments():
    k, v, table, lens = cache()
    scores, positions = torch.zeros((2, 2, 64)), torch.zeros((2, 2, 64), dtype=I32)
    call = lambda s=scores, p=positions, **kw: cache_evict(k, v, table, lens, s, p, **kw)  # noqa: E731
    refuses("budget must be positive", call, budget=0)
    refuses("fit the budget", call, budget=8, first=4, recent=5)
    refuses("fit the budget", call, budget=8, recent=-1)
    refuses("scores must be", call, scores[:, :, :10], budget=8)
    refuses("positions must be", call, scores, scores, budget=8)
    with pytest.raises(AlgxError, match="CUDA tensors only"):
        call(budget=8)


def test_verify_arguments():
    t, d = torch.zeros((2, 4, 9)), torch.zeros((2, 3, 9))
    tok, u, race = torch.zeros((2, 3), dtype=I32), torch.zeros((2, 3)), torch.ones((2, 9))
    call = lambda t=t, tok=tok, d=d, u=u, race=race, **kw: verify_draft(t, tok, d, u, race, **kw)  # noqa: E731
    refuses("mse", call, kind="mse")
    refuses("powers n", call, kind="alg_ce", n=12)
    refuses("positive and finite", call, kind="alg_ce", n=8, c=0.0)
    refuses("temperature is for", call, kind="alg_ce", n=8, c=2.0, temperature=0.5)
    refuses("temperature must be", call, temperature=0.0)
    refuses("at most 31", call, t=torch.zeros((2, 33, 9)))
    refuses("target_logits must have shape", call, t=t[0])
    refuses("bfloat16 or float32", call, t=t.half())
    refuses("draft_logits must have shape", call, d=d.to(BF16))
    refuses("draft_tokens must be", call, tok=tok.long())
    refuses("accept_u must be", call, u=u[:, :2])
    refuses("race must be", call, race=race[:, :8])
    refuses("counts must be", call, counts=torch.zeros(2))
    with pytest.raises(AlgxError, match="CUDA tensors only"):
        call()


def test_c_entries_refuse_without_a_device():
    lib = L.lib()
    cfg = L.PagedConfig(0, 12, 0, 0, 1.0, 1.0)
    none = [None] * 9
    assert lib.algx_paged_attn(cfg, *none, 0, 1, 2, 2, 1, 16, 1, 64, L.ALGX_BF16, None, 0, None) == L.ALGX_ERR_INVALID
    assert b"power of two" in lib.algx_last_error()
    cfg.n = 16
    assert lib.algx_paged_attn(cfg, *none, 1, 1, 2, 2, 1, 16, 1, 64, L.ALGX_BF16, None, 0, None) == L.ALGX_ERR_INVALID
    assert lib.algx_paged_attn(cfg, *none, 0, 1, 2, 2, 1, 16, 1, 64, L.ALGX_BF16, None, 0, None) == L.ALGX_OK
    assert lib.algx_paged_attn(cfg, *none, 0, 1, 2, 2, 1, 24, 1, 64, L.ALGX_BF16, None, 0, None) == L.ALGX_ERR_INVALID
    assert lib.algx_verify_draft(0, 16, 1.0, *[None] * 8, 1, 32, 9, L.ALGX_F32, None) == L.ALGX_ERR_INVALID
    assert lib.algx_cache_evict(*[None] * 6, 4, 3, 2, *[None] * 4, 0, 1, 1, 16, 1, 64, L.ALGX_BF16, None, 0,
                                None) == L.ALGX_ERR_INVALID
    assert b"fit the budget" in lib.algx_last_error()
    assert lib.algx_paged_attn_workspace_size(1, 1, 3, 2, 16, 1, 0, L.ALGX_BF16) == 0
    assert lib.algx_cache_evict_workspace_size(2, 3, 5) >= 2 * 3 * 5 * 4
