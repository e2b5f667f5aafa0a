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


def test_keys_without_a_page_are_refused():
    gen = torch.Generator().manual_seed(1)
    pages = torch.zeros(3, 1, fp4_kv_slab_bytes(16, 64), dtype=torch.uint8)
    q = torch.randn(2, 4, 2, 64, generator=gen)
    lengths = torch.tensor([40, 16], dtype=torch.int32)
    table = torch.tensor([[2, 0, 1], [0, -1, 9]], dtype=torch.int32)  # what no query sees may be anything
    fp4_kv_attention(q, pages, table, lengths)
    for row, column, page in ((0, 2, -1), (0, 0, 3), (1, 0, -1)):
        broken = table.clone()
        broken[row, column] = page
        with pytest.raises(IndexError):
            fp4_kv_attention(q, pages, broken, lengths)
    broken = table.clone()
    broken[0, 0] = -1
    fp4_kv_attention(q, pages, broken, lengths, window=22)  # keys 17 and up
    with pytest.raises(IndexError):
        fp4_kv_attention(q, pages, broken, lengths, window=24)
    with pytest.raises(IndexError):
        fp4_kv_attention(q, pages, table, torch.tensor([49, 1], dtype=torch.int32))
