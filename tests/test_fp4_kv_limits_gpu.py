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
