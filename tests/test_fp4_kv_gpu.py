"""The 4-bit K / V cache's kernels and the page kernels against 64-bit oracles and the CPU
definitions, at the sizes, masks and strides where they can go wrong."""

import pytest
import torch

from tests import _fp4_oracle as oracle

pytestmark = pytest.mark.gpu


def _with_room(table, room, rows):
    """Tables wide enough for ``room`` keys: with many query rows the tensor-core tiles run by then."""
    return torch.nn.functional.pad(table, (0, max(0, -(-room // rows) - table.shape[1])), value=-1)


def _attend_case(cuda, lens, *, h, hk, d, rows, t=1, window=0, sink=None, softcap=None, dtype=torch.bfloat16,
                 qscale=1.0, spread=None, seed=0, one_hot=False, room=0):
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(seed)
    pages, table, lengths = oracle.filled(lens, hk=hk, d=d, rows=rows, gen=gen, device=cuda, spread=spread)
    table = _with_room(table, room, rows)
    q = (qscale * torch.randn(len(lens), h, t, d, generator=gen)).to(cuda, dtype)
    sl = None if sink is None else sink.to(cuda) if torch.is_tensor(sink) else torch.randn(h, generator=gen).to(cuda)
    got = fp4_kv_attention(q, pages, table, lengths, window=window, sink=sl, softcap=softcap)
    check_errors(cuda)
    want, size, score, floor = oracle.attention(q, pages, table, lengths, rows, window=window, sink=sl, softcap=softcap)
    assert got.dtype == dtype and got.shape == q.shape
    err = (got.double() - want).abs()
    if one_hot:  # scores so far apart that one key has all the weight, whatever the scores' error
        score = torch.zeros_like(score)
    allowed = oracle.bound(want, size, score, floor, dtype)
    assert bool((err <= allowed).all()), f"{(err / allowed.clamp(min=1e-300)).max():.3g} of the bound"
    return got


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("rows", [16, 32, 64, 128])
def test_attention_lengths(cuda, d, rows):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 511, 513]
    _attend_case(cuda, lens, h=4, hk=1, d=d, rows=rows, sink=True)
    _attend_case(cuda, lens, h=4, hk=1, d=d, rows=rows, dtype=torch.float16)


@pytest.mark.parametrize("h,hk", [(1, 1), (8, 8), (3, 1), (14, 2), (16, 1), (17, 1), (32, 2), (33, 1), (128, 1)])
def test_attention_head_layouts(cuda, h, hk):
    _attend_case(cuda, [70, 3, 0, 129], h=h, hk=hk, d=64, rows=16, dtype=torch.float16)
    _attend_case(cuda, [70, 3, 0, 129], h=h, hk=hk, d=128, rows=64, sink=True)


@pytest.mark.parametrize("t", [2, 5, 8, 17, 63, 130])
@pytest.mark.parametrize("window", [0, 1, 40])
def test_attention_of_several_tokens(cuda, t, window):
    # lengths below t: the first queries stand before the first key and give zeros
    _attend_case(cuda, [0, 1, t - 1, t, t + 1, 200], h=4, hk=2, d=64, rows=16, t=t, window=window)
    _attend_case(cuda, [t // 2, 150], h=12, hk=1, d=128, rows=32, t=t, window=window, sink=True, dtype=torch.float16)


@pytest.mark.parametrize("window", [1, 15, 16, 33, 128, 1000])
def test_attention_window_and_softcap(cuda, window):
    _attend_case(cuda, [1, 20, 100, 500], h=16, hk=1, d=128, rows=64, window=window, softcap=15.0, qscale=4.0)


@pytest.mark.parametrize("room", [0, 40000])
def test_attention_windows_wider_than_any_cache(cuda, room):
    # less than t keys: the first queries' positions are negative, the window's lower end far below them
    case = dict(h=16, hk=1, d=64, rows=16, t=40, room=room)
    for lens in ([0, 1, 39, 40, 41], [3, 200]):
        want = _attend_case(cuda, lens, **case)
        for window in (2 ** 31 - 1, 2 ** 31 - 20, 2 ** 31):
            assert torch.equal(_attend_case(cuda, lens, window=window, **case), want)


def test_attention_sharp_and_flat_scores(cuda):
    _attend_case(cuda, [300, 1000], h=8, hk=2, d=128, rows=64, qscale=60.0)  # scores in the hundreds
    _attend_case(cuda, [300, 1000], h=8, hk=2, d=128, rows=64, qscale=1e-6)
    _attend_case(cuda, [300], h=8, hk=2, d=128, rows=64, qscale=0.0)
    _attend_case(cuda, [300], h=8, hk=2, d=128, rows=64, qscale=2.0 ** 60, one_hot=True)


def test_attention_sinks_at_the_ends_of_their_type(cuda):
    sink = torch.tensor([float("-inf"), torch.finfo(torch.float32).min, -30.0, 0.0, 30.0, 200.0, -1e4, 1e4])
    _attend_case(cuda, [0, 1, 90, 700], h=8, hk=1, d=64, rows=16, sink=sink)


@pytest.mark.parametrize("spread", [6, 30, 55])
def test_attention_rows_of_very_different_size(cuda, spread):
    """V rows whose scales differ by up to 2^(2 spread): the small ones count when softmax picks them."""
    _attend_case(cuda, [5, 64, 333], h=8, hk=1, d=128, rows=32, spread=spread, qscale=8.0)
    _attend_case(cuda, [5, 64, 333], h=8, hk=2, d=64, rows=16, spread=spread, qscale=30.0)


def test_attention_long_cache_in_splits(cuda):
    _attend_case(cuda, [20000, 7777], h=16, hk=1, d=128, rows=64, sink=True)
    _attend_case(cuda, [9001], h=4, hk=4, d=64, rows=128, dtype=torch.float16)


@pytest.mark.parametrize("room", [0, 1 << 20])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_attention_of_many_rows(cuda, d, dtype, room):
    """Both kernels at the edges of their tiles: 16 rows by 32 keys, and in wide tables 128 by 128."""
    _attend_case(cuda, [128, 129, 300, 0, 39, 1], h=4, hk=2, d=d, rows=16, t=40, dtype=dtype, sink=True, room=room)
    _attend_case(cuda, [700, 256], h=3, hk=1, d=d, rows=48, t=70, dtype=dtype, softcap=12.0, qscale=3.0, room=room)
    _attend_case(cuda, [513, 140], h=16, hk=1, d=d, rows=64, t=9, dtype=dtype, window=100, sink=True,
                 room=room)
    _attend_case(cuda, [3000], h=64, hk=1, d=d, rows=128, t=2, dtype=dtype, room=room)
    _attend_case(cuda, [90, 64, 10], h=4, hk=2, d=d, rows=32, t=20, dtype=dtype, window=30, softcap=9.0, room=room)


@pytest.mark.parametrize("spread", [6, 30, 55])
def test_attention_of_many_rows_of_very_different_size(cuda, spread):
    _attend_case(cuda, [5, 64, 333], h=8, hk=1, d=128, rows=32, t=16, spread=spread, qscale=8.0, room=1 << 20)
    _attend_case(cuda, [260], h=8, hk=2, d=64, rows=16, t=33, spread=spread, qscale=30.0, room=1 << 20)


def test_attention_of_many_rows_sharp_scores(cuda):
    _attend_case(cuda, [300, 200], h=8, hk=1, d=128, rows=64, t=20, qscale=60.0, room=1 << 20)
    _attend_case(cuda, [300], h=8, hk=1, d=64, rows=64, t=20, qscale=0.0, room=1 << 20)
    _attend_case(cuda, [300], h=8, hk=1, d=128, rows=64, t=20, qscale=2.0 ** 60, one_hot=True, room=1 << 20)


def test_attention_of_many_rows_nan_and_bad_pages(cuda):
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention, fp4_kv_write
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(11)
    pages, table, lengths = oracle.filled([200, 180], hk=1, d=128, rows=16, gen=gen, device=cuda)
    table = _with_room(table, 1 << 20, 16)
    q = torch.randn(2, 8, 30, 128, generator=gen).to(cuda, torch.bfloat16)
    clean = fp4_kv_attention(q, pages, table, lengths)
    for which in range(2):
        k, v = torch.randn(2, 1, 1, 128, generator=gen).to(cuda).unbind(0)
        (k, v)[which][0, 0, 40] = float("inf")
        mine = pages.clone()
        fp4_kv_write(k, v, mine, table[0, 195 // 16].long().view(1) * 16 + 195 % 16)  # queries 25 .. 29 see key 195
        got = fp4_kv_attention(q, mine, table, lengths)
        assert bool(got[0, :, 25:].isnan().all() if which == 0 else got[0, :, 25:, 32:64].isnan().all())
        assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :, :25], clean[0, :, :25])
        if which == 1:
            assert bool(got[0, :, 25:, :32].isfinite().all() and got[0, :, 25:, 64:].isfinite().all())
    broken = table.clone()
    broken[0, 3] = 10 ** 6
    out = fp4_kv_attention(q, pages, broken, lengths)
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_errors(cuda)
    assert bool(out.isfinite().all()) and torch.equal(out[1], clean[1])
    # without the keys of that page: the same as a cache in which they were never there
    keep = [i for i in range(200) if i // 16 != 3]
    gathered = torch.zeros_like(pages)
    from saint_llm_b200.ops.fp4_kv import fp4_kv_read

    slots = table[0, torch.tensor(keep, device=cuda) // 16].long() * 16 + torch.tensor(keep, device=cuda) % 16
    k, v = fp4_kv_read(pages, slots, head_dim=128, dtype=torch.float32)
    fp4_kv_write(k, v, gathered, torch.arange(len(keep), device=cuda))
    ids = torch.arange(12, dtype=torch.int32, device=cuda).view(1, 12)
    want, size, score, floor = oracle.attention(q[:1], gathered, ids, torch.tensor([len(keep)], device=cuda), 16)
    assert bool(((out[:1].double() - want).abs() <= oracle.bound(want, size, score, floor, q.dtype)).all())


def test_attention_nan_reaches_only_the_rows_that_see_it(cuda):
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention, fp4_kv_write

    gen = torch.Generator().manual_seed(5)
    pages, table, lengths = oracle.filled([50, 50], hk=1, d=64, rows=16, gen=gen, device=cuda)
    q = torch.randn(2, 4, 3, 64, generator=gen).to(cuda, torch.bfloat16)
    clean = fp4_kv_attention(q, pages, table, lengths)
    for which in range(2):
        k, v = torch.randn(2, 1, 1, 64, generator=gen).to(cuda).unbind(0)
        (k, v)[which][0, 0, 3] = float("nan")
        mine = pages.clone()
        # the last key of sequence 0: only its last query sees it
        fp4_kv_write(k, v, mine, table[0, 49 // 16].long().view(1) * 16 + 49 % 16)
        got = fp4_kv_attention(q, mine, table, lengths)
        seen = got[0, :, 2] if which == 0 else got[0, :, 2, :32]
        assert bool(seen.isnan().all())
        assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :, :2], clean[0, :, :2])


def test_attention_strides_and_streams(cuda):
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention

    gen = torch.Generator().manual_seed(6)
    pages, table, lengths = oracle.filled([100, 37], hk=2, d=64, rows=16, gen=gen, device=cuda)
    q = torch.randn(2, 8, 4, 64, generator=gen).to(cuda, torch.bfloat16)
    want = fp4_kv_attention(q, pages, table, lengths)
    token_major = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(fp4_kv_attention(token_major, pages, table, lengths), want)
    odd = torch.empty(2, 8, 4, 65, device=cuda, dtype=q.dtype)[..., 1:]  # rows off every 16-byte boundary
    odd.copy_(q)
    assert torch.equal(fp4_kv_attention(odd, pages, table, lengths), want)
    layers = torch.empty(pages.shape[0], 3, *pages.shape[1:], dtype=torch.uint8, device=cuda)
    layers[:, 1] = pages
    assert torch.equal(fp4_kv_attention(q, layers[:, 1], table, lengths), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [fp4_kv_attention(q, pages, table, lengths) for _ in range(8)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)
    assert torch.equal(fp4_kv_attention(q[:, :, :1].squeeze(2), pages, table, lengths),
                       fp4_kv_attention(q[:, :, :1], pages, table, lengths).squeeze(2))


def test_attention_in_a_cuda_graph_follows_the_lengths(cuda):
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention

    gen = torch.Generator().manual_seed(8)
    pages, table, lengths = oracle.filled([700, 650], hk=1, d=128, rows=64, gen=gen, device=cuda)
    q = torch.randn(2, 16, 128, generator=gen).to(cuda, torch.bfloat16)
    now = torch.ones_like(lengths)
    fp4_kv_attention(q, pages, table, now)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fp4_kv_attention(q, pages, table, now)
    for n in ([1, 0], [64, 65], [650, 649], [300, 2]):
        now.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, fp4_kv_attention(q, pages, table, now))


def test_attention_pages_past_32_bit_offsets(cuda):
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention, fp4_kv_read, fp4_kv_slab_bytes, fp4_kv_write

    slab = fp4_kv_slab_bytes(64, 128)
    n = 2 ** 32 // slab + 10
    pages = torch.empty(n, 1, slab, dtype=torch.uint8, device=cuda)
    ids = torch.tensor([n - 1, 0, n - 3], device=cuda)
    gen = torch.Generator().manual_seed(9)
    k, v = torch.randn(2, 150, 1, 128, generator=gen).to(cuda).unbind(0)
    pos = torch.arange(150, device=cuda)
    slots = ids[pos // 64] * 64 + pos % 64
    fp4_kv_write(k, v, pages, slots)
    small = torch.empty(3, 1, slab, dtype=torch.uint8, device=cuda)
    fp4_kv_write(k, v, small, pos)
    q = torch.randn(1, 16, 128, generator=gen).to(cuda, torch.bfloat16)
    length = torch.tensor([150], dtype=torch.int32, device=cuda)
    a = fp4_kv_attention(q, pages, ids.int().view(1, 3), length)
    b = fp4_kv_attention(q, small, torch.arange(3, device=cuda).int().view(1, 3), length)
    assert torch.equal(a, b)
    assert all(torch.equal(x, y) for x, y in zip(fp4_kv_read(pages, slots, head_dim=128),
                                                 fp4_kv_read(small, pos, head_dim=128), strict=True))


@pytest.mark.parametrize("n,hk,d,rows", [(1, 1, 128, 64), (37, 2, 64, 16), (1000, 1, 32, 16), (513, 8, 128, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_write_and_read_equal_the_definition(cuda, n, hk, d, rows, dtype):
    from saint_llm_b200.ops import fp4_kv
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(n)
    k = torch.randn(n, hk, d, generator=gen) * 4.0 ** torch.randint(-4, 5, (n, hk, 1), generator=gen)
    v = torch.randint(-48, 49, (n, hk, d), generator=gen) / 8.0  # many ties
    v[0, 0, :32] = 0.0
    v[n // 2, 0, 5] = float("nan")
    k[n // 3, -1, d - 1] = float("inf")
    k, v = k.to(dtype), v.to(dtype)
    pages = torch.randint(0, 256, (-(-n // rows) + 1, hk, fp4_kv.fp4_kv_slab_bytes(rows, d)), generator=gen,
                          dtype=torch.uint8)
    slots = torch.randperm(pages.shape[0] * rows, generator=gen)[:n]
    if n > 1:
        slots[-1] = -1
    mine = pages.to(cuda)
    fp4_kv.fp4_kv_write(k, v, pages, slots)
    fp4_kv.fp4_kv_write(k.to(cuda), v.to(cuda), mine, slots.to(cuda))
    check_errors(cuda)
    assert torch.equal(mine.cpu(), pages)
    for out in (torch.bfloat16, torch.float16, torch.float32):
        for a, b in zip(fp4_kv.fp4_kv_read(mine, slots.to(cuda), head_dim=d, dtype=out),
                        fp4_kv.fp4_kv_read(pages, slots, head_dim=d, dtype=out), strict=True):
            assert torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))


def test_write_fp32_next_to_ties(cuda):
    """Values one unit in the last place from every rounding boundary, at several scales."""
    from saint_llm_b200.ops import fp4_kv

    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = torch.cat([ties, torch.nextafter(ties, torch.tensor(9.0)), torch.nextafter(ties, torch.tensor(0.0))])
    row = torch.cat([near, torch.tensor([6.0]), -near[:10]]) * 2.0 ** torch.tensor([[-20.0], [0.0], [3.0], [40.0]])
    row = row.view(1, 1, 128)
    edge = torch.tensor([[3.0, 6.0], [1.5, 0.75]]).view(-1)  # amax at, just above and just below 6 * 2^e
    amax = torch.stack([edge, torch.nextafter(edge, torch.tensor(9.0)), torch.nextafter(edge, torch.tensor(0.0)), edge])
    other = torch.zeros(1, 1, 4, 32)
    other[0, 0, :, 0] = amax[:, 1]
    other[0, 0, :, 1] = amax[:, 0] / 3
    other = other.view(1, 1, 128)
    a = torch.zeros(1, 1, fp4_kv.fp4_kv_slab_bytes(16, 128), dtype=torch.uint8)
    b = a.to(cuda)
    fp4_kv.fp4_kv_write(row, other, a, torch.tensor([3]))
    fp4_kv.fp4_kv_write(row.to(cuda), other.to(cuda), b, torch.tensor([3], device=cuda))
    assert torch.equal(b.cpu(), a)


def test_write_takes_strided_rows(cuda):
    from saint_llm_b200.ops import fp4_kv

    gen = torch.Generator().manual_seed(2)
    qkv = torch.randn(20, 5, 64, generator=gen).to(cuda, torch.bfloat16)
    pages = torch.zeros(2, 2, fp4_kv.fp4_kv_slab_bytes(16, 64), dtype=torch.uint8, device=cuda)
    want = pages.clone()
    slots = torch.arange(20, device=cuda)
    fp4_kv.fp4_kv_write(qkv[:, 1:3].contiguous(), qkv[:, 3:5].contiguous(), want, slots)
    fp4_kv.fp4_kv_write(qkv[:, 1:3], qkv[:, 3:5], pages, slots)
    assert torch.equal(pages, want)
    odd = torch.empty(20, 2, 67, device=cuda, dtype=torch.bfloat16)[..., 2:66]
    odd.copy_(qkv[:, 1:3])
    pages.zero_()
    fp4_kv.fp4_kv_write(odd, qkv[:, 3:5], pages, slots)
    assert torch.equal(pages, want)


def test_indexes_outside_are_recorded_and_skipped(cuda):
    from saint_llm_b200.ops import fp4_kv
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(4)
    pages, table, lengths = oracle.filled([40], hk=1, d=64, rows=16, gen=gen, device=cuda)
    before = pages.clone()
    row = torch.randn(1, 1, 64, device=cuda)
    for slot in (pages.shape[0] * 16, -2):
        fp4_kv.fp4_kv_write(row, row, pages, torch.tensor([slot], device=cuda))
        with pytest.raises(RuntimeError, match="out of bounds"):
            check_errors(cuda)
        assert torch.equal(pages, before)
    assert not fp4_kv.fp4_kv_read(pages, torch.tensor([10 ** 9], device=cuda), head_dim=64)[0].any()
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_errors(cuda)
    q = torch.randn(1, 4, 64, device=cuda, dtype=torch.bfloat16)
    for bad in (10 ** 6, -1):
        broken = table.clone()
        broken[0, 1] = bad
        out = fp4_kv.fp4_kv_attention(q, pages, broken, lengths)
        with pytest.raises(RuntimeError, match="out of bounds"):
            check_errors(cuda)
        assert bool(out.isfinite().all())
    out = fp4_kv.fp4_kv_attention(q, pages, table, torch.tensor([10 ** 6], dtype=torch.int32, device=cuda))
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_errors(cuda)
    negative = fp4_kv.fp4_kv_attention(q, pages, table, torch.tensor([-5], dtype=torch.int32, device=cuda))
    assert not negative.any()
    check_errors(cuda)


def test_refusals(cuda):
    from saint_llm_b200.ops import fp4_kv
    from saint_llm_b200.ops.pages import compact_pages, fork_pages

    pages = torch.zeros(2, 1, fp4_kv.fp4_kv_slab_bytes(16, 64), dtype=torch.uint8, device=cuda)
    table = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    lengths = torch.ones(1, dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device=cuda)
    bad = [(q.float(), pages, table, lengths, {}), (q[..., :48], pages, table, lengths, {}),
           (q, pages[..., :-8], table, lengths, {}), (q, pages.float(), table, lengths, {}),
           (q, pages.cpu(), table, lengths, {}), (q, pages, table.long(), lengths, {}),
           (q, pages, table, lengths.long(), {}), (q, pages, table.cpu(), lengths, {}),
           (q, pages.expand(2, 3, -1), table, lengths, {}), (q, pages, table, lengths, {"window": -1}),
           (q, pages, table, lengths, {"softcap": -1.0}), (q, pages, table, lengths, {"sink": q[0, :3, 0, 0]}),
           (q, pages, table.expand(2, -1), lengths, {})]
    for a, b, c, e, kw in bad:
        with pytest.raises(RuntimeError):
            fp4_kv.fp4_kv_attention(a, b, c, e, **kw)
    row, slot = torch.zeros(1, 1, 64, device=cuda), torch.zeros(1, dtype=torch.long, device=cuda)
    for k, v, p, s in [(row, row.half(), pages, slot), (row, row, pages, slot.int()), (row.long(), row.long(), pages, slot),
                       (row.expand(1, 2, 64), row.expand(1, 2, 64), pages, slot), (row.cpu(), row.cpu(), pages, slot),
                       (row.expand(2, 1, 64), row.expand(2, 1, 64), pages, slot)]:
        with pytest.raises(RuntimeError):
            fp4_kv.fp4_kv_write(k, v, p, s)
    pool, refs = torch.zeros(2, 8, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    one = torch.zeros(1, dtype=torch.int32, device=cuda)
    for args in [(pool[:, :6], table, lengths, refs, one, one), (pool, table.long(), lengths, refs, one, one),
                 (pool, table, lengths, refs[:1], one, one), (pool, table, lengths, refs, one, one.long()),
                 (pool, table, lengths, refs, one.expand(2), one), (pool.cpu(), table, lengths, refs, one, one)]:
        with pytest.raises((RuntimeError, ValueError)):
            fork_pages(*args, page_rows=4)
    with pytest.raises(RuntimeError):
        fork_pages(pool, table, lengths, refs, one, one, page_rows=0)
    with pytest.raises(RuntimeError):
        compact_pages(pool[:, :6], table, refs)
    # nothing to do is no error
    assert fp4_kv.fp4_kv_attention(q[:0], pages, table[:0], lengths[:0]).shape == (0, 4, 1, 64)
    fp4_kv.fp4_kv_write(row[:0], row[:0], pages, slot[:0])
    assert fp4_kv.fp4_kv_read(pages, slot[:0], head_dim=64)[0].shape == (0, 1, 64)


# ----------------------------------------------------------------------------- pages
def _pool(n_pages, dim, dtype, gen):
    x = torch.randint(-100, 100, (n_pages, dim), generator=gen)
    return x.to(dtype)


def _table(seqs, width, rows, n_pages, gen):
    lens = torch.randint(0, width * rows + 1, (seqs,), generator=gen).tolist()
    order = torch.randperm(n_pages, generator=gen).tolist()
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    for i in range(seqs):
        lens[i] = min(lens[i], max(0, (len(order) - seqs) * rows))
        for c in range(-(-lens[i] // rows)):
            table[i, c] = order.pop()
            refs[table[i, c]] += 1
    return table, torch.tensor(lens, dtype=torch.int32), refs


@pytest.mark.parametrize("seqs,width,rows,n_pages,dim,dtype", [
    (1, 1, 16, 3, 16, torch.bfloat16), (7, 5, 4, 60, 48, torch.float32), (40, 9, 16, 700, 4096, torch.uint8),
    (300, 3, 64, 3000, 136, torch.bfloat16), (1100, 2, 8, 5000, 16, torch.uint8)])
def test_fork_equals_the_definition(cuda, seqs, width, rows, n_pages, dim, dtype):
    from saint_llm_b200.ops.gemm import check_errors
    from saint_llm_b200.ops.pages import fork_pages

    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        pool = _pool(n_pages, dim, dtype, gen)
        table, lengths, refs = _table(seqs, width, rows, n_pages, gen)
        n = max(1, seqs if seed == 2 else seqs // 2)
        children = torch.randperm(seqs, generator=gen)[:n].int()
        parents = torch.randint(-1, seqs, (n,), generator=gen).int()
        mine = pool.to(cuda)
        got = fork_pages(mine, *(x.to(cuda) for x in (table, lengths, refs, parents, children)), page_rows=rows)
        want = fork_pages(pool, table, lengths, refs, parents, children, page_rows=rows)
        check_errors(cuda)
        for a, b in zip(got, want, strict=True):
            assert torch.equal(a.cpu(), b)
        assert torch.equal(mine.cpu(), pool)


def test_fork_without_room_changes_nothing(cuda):
    from saint_llm_b200.ops.gemm import check_errors
    from saint_llm_b200.ops.pages import fork_pages

    pool = torch.randn(3, 8, device=cuda)
    table = torch.tensor([[0, 1], [-1, -1], [-1, -1]], dtype=torch.int32, device=cuda)
    lengths = torch.tensor([5, 0, 0], dtype=torch.int32, device=cuda)
    refs = torch.tensor([1, 1, 0], dtype=torch.int32, device=cuda)
    both = torch.tensor([1, 2], dtype=torch.int32, device=cuda)
    keep = pool.clone()
    got = fork_pages(pool, table, lengths, refs, torch.zeros_like(both), both, page_rows=4)
    with pytest.raises(RuntimeError, match="no free page"):
        check_errors(cuda)
    assert torch.equal(pool, keep)
    assert all(torch.equal(a, b) for a, b in zip(got, (table, lengths, refs), strict=True))
    # a fork of a row that does not exist is skipped
    got = fork_pages(pool, table, lengths, refs, both + 8, both, page_rows=4)
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_errors(cuda)
    assert all(torch.equal(a, b) for a, b in zip(got, (table, lengths, refs), strict=True))


@pytest.mark.parametrize("seqs,width,n_pages,dim,dtype", [
    (1, 1, 1, 16, torch.uint8), (7, 5, 60, 24, torch.float32), (40, 9, 1024, 4096, torch.uint8),
    (300, 3, 3001, 8, torch.bfloat16)])
def test_compact_equals_the_definition(cuda, seqs, width, n_pages, dim, dtype):
    from saint_llm_b200.ops.gemm import check_errors
    from saint_llm_b200.ops.pages import compact_pages

    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        pool = _pool(n_pages, dim, dtype, gen)
        table, _, refs = _table(seqs, width, 4, n_pages, gen)
        if seed == 1:  # rows that share pages, and rows that are gone
            table[seqs // 2] = table[0]
            table[seqs - 1] = -1
            refs = torch.bincount(table[table >= 0].long(), minlength=n_pages).int()
        if seed == 2:
            table.fill_(-1)
            refs.zero_()
        mine = pool.to(cuda)
        got = compact_pages(mine, table.to(cuda), refs.to(cuda))
        want = compact_pages(pool, table, refs)
        check_errors(cuda)
        for a, b in zip(got, want, strict=True):
            assert torch.equal(a.cpu(), b)
        n = int(want[2])
        assert torch.equal(mine[:n].cpu(), pool[:n])


def test_page_kernels_on_a_pool_past_32_bit_offsets(cuda):
    from saint_llm_b200.ops.pages import compact_pages, fork_pages

    size = 1 << 20
    pool = torch.empty(4200, size, dtype=torch.uint8, device=cuda)
    pool[4199] = torch.arange(size, device=cuda).to(torch.uint8)
    want = pool[4199].clone()
    refs = torch.ones(4200, dtype=torch.int32, device=cuda)
    refs[4198] = 0
    table = torch.tensor([[4199], [-1]], dtype=torch.int32, device=cuda)
    lengths = torch.tensor([3, 0], dtype=torch.int32, device=cuda)
    zero, one = torch.zeros(1, dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda)
    t2, _, _ = fork_pages(pool, table, lengths, refs, zero, one, page_rows=4)
    assert int(t2[1, 0]) == 4198 and torch.equal(pool[4198], want)
    pool[4198].zero_()
    t3, _, n = compact_pages(pool, table, refs)
    assert int(n) == 4199 and int(t3[0, 0]) == 4198 and torch.equal(pool[4198], want)
