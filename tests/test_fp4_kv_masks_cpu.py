"""The CPU definition of attention on the 4-bit cache: what a query does not see does not reach it."""

import pytest
import torch

from saint_llm_b200.ops.fp4_kv import fp4_kv_attention, fp4_kv_slab_bytes, fp4_kv_write


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("hk", [1, 2])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_nan_blocks_reach_only_the_queries_that_see_them(which, hk, value):
    gen = torch.Generator().manual_seed(0)
    pages = torch.zeros(2, hk, fp4_kv_slab_bytes(16, 64), dtype=torch.uint8)
    k, v = torch.randn(2, 20, hk, 64, generator=gen).unbind(0)
    slots, table = torch.arange(20), torch.tensor([[0, 1]], dtype=torch.int32)
    lengths = torch.tensor([20], dtype=torch.int32)
    q = torch.randn(1, 4, 5, 64, generator=gen)
    fp4_kv_write(k, v, pages, slots)
    clean = fp4_kv_attention(q, pages, table, lengths, window=6)
    assert bool(clean.isfinite().all())
    # queries stand at 15 .. 19 and see six keys each: key 12 reaches 15 .. 17, key 19 the last one
    for key, seen in ((12, slice(0, 3)), (19, slice(4, 5))):
        mine, x = pages.clone(), {"k": k.clone(), "v": v.clone()}
        x[which][key, hk - 1, 3] = value
        fp4_kv_write(x["k"], x["v"], mine, slots)
        got = fp4_kv_attention(q, mine, table, lengths, window=6)
        heads = slice(4 - 4 // hk, 4)  # those that read the last K / V head
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[:, heads, seen, :64 if which == "k" else 32] = True
        assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], clean[~hit])
