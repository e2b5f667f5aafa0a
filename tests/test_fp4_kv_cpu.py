"""The 4-bit K / V cache's definitions against a 64-bit oracle, the page operators' invariants,
and refusals (no GPU)."""

import numpy as np
import pytest
import torch

from saint_llm_b200.infer.paged_kv import PoolExhausted
from saint_llm_b200.ops import fp4_kv
from saint_llm_b200.ops.pages import compact_pages, fork_pages
from tests import _fp4_oracle as oracle


@pytest.mark.parametrize("d,rows,dtype", [(32, 16, torch.float32), (64, 16, torch.bfloat16), (128, 32, torch.float16)])
def test_write_is_byte_for_byte_the_format(d, rows, dtype):
    gen = torch.Generator().manual_seed(d)
    k = torch.randn(5, 2, d, generator=gen) * 10.0 ** torch.randint(-3, 4, (5, 2, 1), generator=gen)
    v = torch.randn(5, 2, d, generator=gen)
    v[0, 0, :32] = 0.0                                    # a block of zeros
    v[1, 0, 0] = 6.0 * 2.0 ** 3                           # amax exactly 6 * 2^e
    v[2, 0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])  # every tie
    v[2, 0, 8:32] = 0.0
    v[3, 1, 3] = float("nan")
    v[4, 1, 5] = float("-inf")
    k, v = k.to(dtype), v.to(dtype)
    pages = torch.randint(0, 256, (3, 2, fp4_kv.fp4_kv_slab_bytes(rows, d)), generator=gen, dtype=torch.uint8)
    want = pages.numpy().copy()
    slots = torch.tensor([2 * rows + 1, 0, rows - 1, 2 * rows, rows])
    fp4_kv.fp4_kv_write(k, v, pages, slots)
    for i, s in enumerate(slots.tolist()):
        vi = v[i].double().numpy()
        oracle.put(want, rows, s, k[i].double().numpy(), vi)
    # where the scale says NaN the codes carry nothing
    assert np.array_equal(pages.numpy(), want)
    got = fp4_kv.fp4_kv_read(pages, slots, head_dim=d, dtype=torch.float32)
    for x, y in ((k, got[0]), (v, got[1])):
        assert np.array_equal(oracle.quantise(x.double().numpy())[2], y.double().numpy(), equal_nan=True)


def test_write_skips_and_read_zeros():
    gen = torch.Generator().manual_seed(0)
    pages = torch.randint(0, 256, (2, 1, fp4_kv.fp4_kv_slab_bytes(16, 32)), generator=gen, dtype=torch.uint8)
    before = pages.clone()
    k = torch.randn(2, 1, 32, generator=gen)
    fp4_kv.fp4_kv_write(k, k, pages, torch.tensor([-1, -1]))
    assert torch.equal(pages, before)
    got, _ = fp4_kv.fp4_kv_read(pages, torch.tensor([-1]), head_dim=32)
    assert got.dtype == torch.bfloat16 and not got.any()


@pytest.mark.parametrize("t,window,sink,softcap,lens", [
    (1, 0, False, None, [0, 1, 17, 40]), (1, 5, True, None, [0, 1, 33]), (3, 0, True, 20.0, [1, 2, 3, 50]),
    (4, 7, False, None, [0, 2, 9, 31])])
def test_attention_definition(t, window, sink, softcap, lens):
    gen = torch.Generator().manual_seed(7)
    pages, table, lengths = oracle.filled(lens, hk=2, d=32, rows=16, gen=gen, device="cpu")
    q = torch.randn(len(lens), 6, t, 32, generator=gen, dtype=torch.float64)
    sl = torch.randn(6, generator=gen) if sink else None
    got = fp4_kv.fp4_kv_attention(q, pages, table, lengths, window=window, sink=sl, softcap=softcap)
    want, *_ = oracle.attention(q, pages, table, lengths, 16, window=window, sink=sl, softcap=softcap)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-13)
    assert not got[:, :, 0][lengths < t].any()  # those queries stand before the first key


def test_three_dimensional_q_is_one_token():
    gen = torch.Generator().manual_seed(3)
    pages, table, lengths = oracle.filled([9], hk=1, d=64, rows=16, gen=gen, device="cpu")
    q = torch.randn(1, 4, 64, generator=gen)
    a = fp4_kv.fp4_kv_attention(q, pages, table, lengths)
    b = fp4_kv.fp4_kv_attention(q.unsqueeze(2), pages, table, lengths)
    assert a.shape == q.shape and torch.equal(a, b.squeeze(2))


def test_refusals():
    pages = torch.zeros(2, 1, fp4_kv.fp4_kv_slab_bytes(16, 32), dtype=torch.uint8)
    row = torch.zeros(1, 1, 32)
    for slots in (torch.tensor([32]), torch.tensor([-2])):
        with pytest.raises(IndexError):
            fp4_kv.fp4_kv_write(row, row, pages, slots)
        with pytest.raises(IndexError):
            fp4_kv.fp4_kv_read(pages, slots, head_dim=32)
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_write(row, row.half(), pages, torch.tensor([0]))
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_write(row, row, pages, torch.tensor([0], dtype=torch.int32))
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_slab_bytes(24, 64)
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_slab_bytes(16, 96)
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_page_rows(torch.zeros(1, 1, 100, dtype=torch.uint8), 32)
    q, table, lengths = torch.zeros(1, 3, 1, 32), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_attention(q, pages, table.long(), lengths)
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_attention(q, pages, table, lengths, window=-1)
    with pytest.raises(ValueError):
        fp4_kv.fp4_kv_attention(q, torch.zeros(2, 2, pages.shape[2], dtype=torch.uint8), table, lengths)
    pool, refs = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        fork_pages(pool, table, lengths.view(1), refs, torch.tensor([0]), torch.tensor([0, 0]), page_rows=4)
    with pytest.raises(ValueError):
        compact_pages(pool, table, refs[:1])
    with pytest.raises(IndexError):
        fork_pages(pool, table, lengths, refs, torch.tensor([3]), torch.tensor([0]), page_rows=4)


# ----------------------------------------------------------------------------- pages
def _state(gen, seqs=6, width=5, rows=4, n_pages=40, dim=3):
    pool = torch.randn(n_pages, rows, dim, generator=gen)
    lens = torch.randint(0, width * rows + 1, (seqs,), generator=gen).tolist()
    order = torch.randperm(n_pages, generator=gen).tolist()
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    for i, n in enumerate(lens):
        for c in range(-(-n // rows)):
            table[i, c] = order.pop()
            refs[table[i, c]] += 1
    return pool, table, torch.tensor(lens, dtype=torch.int32), refs


def _contents(pool, table, lengths):
    out = []
    for row, n in zip(table.tolist(), lengths.tolist(), strict=True):
        pages = [p for p in row if p >= 0]
        flat = pool[pages].reshape(-1, pool.shape[-1]) if pages else pool.new_zeros(0, pool.shape[-1])
        out.append(flat[:n].clone())
    return out


def _counts(table, n_pages):
    return torch.bincount(table[table >= 0].long(), minlength=n_pages).int()


@pytest.mark.parametrize("seed", range(6))
def test_fork_keeps_contents_and_counts(seed):
    gen = torch.Generator().manual_seed(seed)
    pool, table, lengths, refs = _state(gen)
    before = _contents(pool, table, lengths)
    children = torch.randperm(6, generator=gen)[:4].int()
    parents = torch.randint(-1, 6, (4,), generator=gen).int()
    t2, l2, r2 = fork_pages(pool, table, lengths, refs, parents, children, page_rows=4)
    after = _contents(pool, t2, l2)
    source = {c: p for p, c in zip(parents.tolist(), children.tolist(), strict=True)}
    for i in range(6):
        p = source.get(i, i)
        assert torch.equal(after[i], before[p] if p >= 0 else before[0][:0])
    assert torch.equal(_counts(t2, 40), r2)
    # a partly filled last page has one holder, unless its row was left as it was
    for i in source:
        if source[i] not in (-1, i) and l2[i] % 4:
            assert r2[t2[i, l2[i] // 4]] == 1


def test_fork_then_free_returns_every_page():
    gen = torch.Generator().manual_seed(1)
    pool, table, lengths, refs = _state(gen)
    every = torch.arange(6, dtype=torch.int32)
    table, lengths, refs = fork_pages(pool, table, lengths, refs, torch.zeros(6, dtype=torch.int32), every, page_rows=4)
    table, lengths, refs = fork_pages(pool, table, lengths, refs, torch.full((6,), -1, dtype=torch.int32), every,
                                      page_rows=4)
    assert not refs.any() and (table == -1).all() and not lengths.any()


def test_fork_without_room_changes_nothing():
    pool = torch.randn(2, 4, 1)
    keep = pool.clone()
    table = torch.tensor([[0, 1], [-1, -1]], dtype=torch.int32)
    with pytest.raises(PoolExhausted):
        fork_pages(pool, table, torch.tensor([5, 0], dtype=torch.int32), torch.tensor([1, 1], dtype=torch.int32),
                   torch.tensor([0]), torch.tensor([1]), page_rows=4)
    assert torch.equal(pool, keep)


@pytest.mark.parametrize("seed", range(6))
def test_compact_keeps_contents(seed):
    gen = torch.Generator().manual_seed(seed)
    pool, table, lengths, refs = _state(gen)
    table, lengths, refs = fork_pages(pool, table, lengths, refs, torch.tensor([0, -1]), torch.tensor([1, 2]), page_rows=4)
    before = _contents(pool, table, lengths)
    t2, r2, n = compact_pages(pool, table, refs)
    assert int(n) == int((refs > 0).sum()) and (r2[:n] > 0).all() and not r2[n:].any()
    assert torch.equal(_counts(t2, 40), r2)
    assert all(torch.equal(a, b) for a, b in zip(before, _contents(pool, t2, lengths), strict=True))
