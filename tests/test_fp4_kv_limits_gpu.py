"""The 4-bit K / V cache's kernels at the ends of their ranges: sizes past 32 bits, values near the
ends of fp32, scores that leave no room for fractions."""

import pytest
import torch

from tests import _fp4_oracle as oracle

pytestmark = pytest.mark.gpu


def test_pages_longer_than_31_bits(cuda):
    """The last head's slab of a page of 2.2 GB lies past 2^31 bytes."""
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention, fp4_kv_read, fp4_kv_slab_bytes, fp4_kv_write
    from saint_llm_b200.ops.gemm import check_errors

    rows, heads = 65536, 250
    pages = torch.zeros(1, heads, fp4_kv_slab_bytes(rows, 128), dtype=torch.uint8, device=cuda)
    gen = torch.Generator().manual_seed(1)
    k, v = torch.randint(-3, 4, (2, 5, heads, 128), generator=gen).to(cuda, torch.bfloat16).unbind(0)
    slots = torch.tensor([0, 1, 17, 40000, rows - 1], device=cuda)
    fp4_kv_write(k, v, pages, slots)
    check_errors(cuda)
    back = fp4_kv_read(pages, slots, head_dim=128)
    check_errors(cuda)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    q = torch.randn(1, heads, 1, 128, generator=gen).to(cuda, torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32, device=cuda)
    assert torch.equal(fp4_kv_attention(q, pages, torch.zeros(1, 1, dtype=torch.int32, device=cuda), one)[0, :, 0], v[0])
    check_errors(cuda)


def test_reserve_where_lengths_and_a_page_pass_31_bits(cuda):
    from saint_llm_b200.ops.gemm import check_errors
    from saint_llm_b200.ops.pages import reserve_rows

    rows = 2 ** 30 - 1
    table = torch.tensor([[4, -1]], dtype=torch.int32, device=cuda)
    lengths = torch.tensor([rows], dtype=torch.int32, device=cuda)  # the first page is full
    refs = torch.tensor([1, 0, 1, 1, 1], dtype=torch.int32, device=cuda)
    slots = reserve_rows(table, lengths, refs, torch.zeros(1, dtype=torch.int32, device=cuda), 3, page_rows=rows)
    check_errors(cuda)
    assert slots.tolist() == [[rows, rows + 1, rows + 2]]
    assert table.tolist() == [[4, 1]] and lengths.tolist() == [rows + 3] and refs.tolist() == [1] * 5


def test_more_pages_than_32_bits_count_are_refused(cuda):
    from saint_llm_b200.ops.pages import compact_pages, fork_pages, reserve_rows

    n = 2 ** 31 - 100
    refs = torch.empty(n, dtype=torch.int32, device=cuda)
    pool = torch.empty(n, 0, device=cuda)
    table, one = (torch.zeros(s, dtype=torch.int32, device=cuda) for s in ((1, 1), (1,)))
    with pytest.raises(RuntimeError, match="32 bits"):
        compact_pages(pool, table, refs)
    with pytest.raises(RuntimeError, match="32 bits"):
        fork_pages(pool, table, one, refs, one, one, page_rows=4)
    with pytest.raises(RuntimeError, match="32 bits"):
        reserve_rows(table, one, refs, one, 1, page_rows=4)
