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


# ----------------------------------------------------------------------------- attention
BOTH = pytest.mark.parametrize("room", [0, 1 << 20], ids=["few_rows", "many_rows"])


def _cache(cuda, k, v, rows, room):
    """Pages with the rows k, v (N, heads, d) fp32 of one sequence, and a table wide enough for ``room`` keys
    (with many query rows the tensor-core tiles run by then)."""
    from saint_llm_b200.ops.fp4_kv import fp4_kv_slab_bytes, fp4_kv_write

    n, hk, d = k.shape
    count = -(-n // rows)
    pages = torch.zeros(count, hk, fp4_kv_slab_bytes(rows, d), dtype=torch.uint8, device=cuda)
    fp4_kv_write(k.to(cuda), v.to(cuda), pages, torch.arange(n, device=cuda))
    table = torch.full((1, max(count, -(-room // rows))), -1, dtype=torch.int32, device=cuda)
    table[0, :count] = torch.arange(count, dtype=torch.int32, device=cuda)
    return pages, table, torch.tensor([n], dtype=torch.int32, device=cuda)


def _definition(q, k, v, *, window=0, softcap=None, scale):
    """(out, size, score, floor) in 64 bits, as the oracle's, for one sequence and K / V head; all of them by
    dim: what a dim may be off by depends on that dim's values alone."""
    _, h, t, d = q.shape
    n = len(k)
    pos = torch.arange(n - t, n, device=q.device).view(1, t, 1)
    key = torch.arange(n, device=q.device)
    seen = (key <= pos) & ((key > pos - window) if window else True)
    k, v = k[:, 0], v[:, 0]
    s = torch.einsum("htd,nd->htn", q[0].double(), k) * scale
    size = torch.einsum("htd,nd->htn", q[0].double().abs(), k.abs()) * abs(scale)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = torch.where(seen, s, float("-inf"))
    p = torch.softmax(s, -1)
    score = torch.where(p > 2.0 ** -45, size, 0.0).amax(-1, keepdim=True)  # an error matters where there is weight
    floor = (torch.where(seen.unsqueeze(-1), v.abs(), 0.0).amax(2) * seen.sum(-1, keepdim=True)).expand(h, t, d)
    return p @ v, p @ v.abs(), score, floor


def _check(cuda, k, v, q, *, rows=32, room=0, extra=0.0, scale=1.0, blunt=False, **kw):
    """k, v (N, 1, d) fp32, q (1, H, T, d) in 16 bits."""
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention
    from saint_llm_b200.ops.gemm import check_errors

    pages, table, lengths = _cache(cuda, k, v, rows, room)
    q = q.to(cuda)
    got = fp4_kv_attention(q, pages, table, lengths, scale=scale, **kw)[0]
    check_errors(cuda)
    kk, vv = oracle.rows_of(pages, rows, q.shape[-1], torch.arange(len(k), device=cuda))
    want, size, score, floor = _definition(q, kk, vv, scale=scale, **kw)
    if blunt:  # scores so far apart, or V so alike, that the scores' own rounding does not show
        score = torch.zeros_like(score)
    allowed = oracle.bound(want, size, score, floor, q.dtype) + extra
    err = (got.double() - want).abs()
    assert bool((err <= allowed).all()), \
        f"{float((err / allowed).nan_to_num(float('inf')).max()):.3g} of the bound, {int((~(err <= allowed)).sum())} of {err.numel()}"


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen)


@BOTH
@pytest.mark.parametrize("softcap", [None, 1e9])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_up_to_2_28_keep_their_weights(cuda, room, sign, softcap):
    """Scores with no room for fractions, a unit or so apart within and between tiles.  All keys have
    the same V, so whatever the weights, the output is V."""
    gen = torch.Generator().manual_seed(3)
    for low in (15, 20, 22, 24, 26):
        q = torch.zeros(1, 16, 20, 64)
        q[..., 0] = sign * 2.0 ** (low + 2 * torch.rand(1, 16, 20, generator=gen))
        q[..., 1] = 0.2 + 1.6 * torch.rand(1, 16, 20, generator=gen)
        k = torch.zeros(400, 1, 64)
        k[:, 0, 0] = 1.0
        k[:, 0, 1] = torch.randint(0, 3, (400,), generator=gen)
        k[torch.randperm(400, generator=gen)[:100], 0, 0] = 0.5
        v = torch.randint(1, 5, (1, 1, 64), generator=gen).float().expand(400, 1, 64)
        _check(cuda, k, v, q.bfloat16(), room=room, softcap=softcap, blunt=True)
        for n in (1, 2, 33, 129):
            _check(cuda, k[:n], v[:n], q[:, :, :1].bfloat16(), softcap=softcap, blunt=True)


@BOTH
@pytest.mark.parametrize("size", [1e-37, 2e-35, 3e-26, 3e-20])
def test_values_down_to_the_smallest_scales(cuda, room, size):
    """Scale bytes down to 2, alone and beside blocks and keys of other sizes."""
    gen = torch.Generator().manual_seed(4)
    for d, tiny in ((128, None), (64, 1e-37), (128, 2e-35)):
        v = size * _rand(gen, 150, 1, d)
        if tiny is not None:
            v[:, :, 32:64] *= tiny / size
            v[7, 0, :32] *= tiny / size
        _check(cuda, _rand(gen, 150, 1, d), v, (0.3 * _rand(gen, 1, 8, 9, d)).bfloat16(), room=room)


@BOTH
def test_blocks_of_the_smallest_scale_are_no_zeros(cuda, room):
    """Scale byte 1: magnitudes up to 6 * 2^-126, which a block of zeros has too."""
    gen = torch.Generator().manual_seed(5)
    small = lambda *shape: torch.randint(-6, 7, shape, generator=gen) * 2.0 ** -126  # noqa: E731
    for d in (64, 128):
        q = (0.3 * _rand(gen, 1, 8, 9, d)).bfloat16()
        v = small(100, 1, d)
        _check(cuda, _rand(gen, 100, 1, d), v, q, room=room)
        q = torch.zeros(1, 8, 9, d)
        q[..., 5], q[..., 40] = 2.0 ** 125 * torch.randint(-3, 4, (2, 1, 8, 9), generator=gen)
        _check(cuda, small(100, 1, d), _rand(gen, 100, 1, d), q.bfloat16(), room=room)


@BOTH
def test_blocks_of_the_smallest_scale_beside_ordinary_ones(cuda, room):
    gen = torch.Generator().manual_seed(12)
    for d in (64, 128):
        q, v = (0.3 * _rand(gen, 1, 8, 9, d)).bfloat16(), _rand(gen, 100, 1, d)
        v[:, :, 32:64] = torch.randint(-6, 7, (100, 1, 32), generator=gen) * 2.0 ** -126
        v[50:, :, :32] = 0.0
        _check(cuda, _rand(gen, 100, 1, d), v, q, room=room)


@BOTH
@pytest.mark.parametrize("size", [2.0 ** -45, 2.0 ** -100, 2.0 ** 60])
def test_keys_of_other_sizes_in_part_filled_tiles(cuda, room, size):
    """What lies beside the keys of a tile has no say in their unit."""
    gen = torch.Generator().manual_seed(13)
    for n in (2, 31, 100):
        q = (_rand(gen, 1, 8, 9 if n > 9 else 2, 64) / size).bfloat16()
        k = size * _rand(gen, n, 1, 64)
        _check(cuda, k, _rand(gen, n, 1, 64), q, room=room)
        _check(cuda, k, _rand(gen, n, 1, 64), q[:, :, -1:], window=20)


@BOTH
@pytest.mark.parametrize("apart", [50, 80, 120, 160])
def test_blocks_of_v_of_very_different_size(cuda, room, apart):
    """Each block of 32 dims is as near as if it were alone, whatever the others' and the other keys' size."""
    gen = torch.Generator().manual_seed(6)
    for d in (64, 128):
        q, k = (0.3 * _rand(gen, 1, 8, 9, d)).bfloat16(), _rand(gen, 300, 1, d)
        v = _rand(gen, 300, 1, d)
        v[:, :, :32] *= 2.0 ** (apart // 2)
        v[:, :, -32:] *= 2.0 ** -((apart + 1) // 2)
        _check(cuda, k, v, q, room=room)
        v = _rand(gen, 300, 1, d) * 2.0 ** torch.randint(-apart // 2, apart // 2 + 1, (300, d // 32), generator=gen) \
            .repeat_interleave(32, -1).view(300, 1, d)
        _check(cuda, k, v, (40 * q.float()).bfloat16(), room=room)


@BOTH
def test_values_at_the_type_s_end_reach_only_the_rows_that_see_them(cuda, room):
    """Keys that earlier rows of the same tile see and later ones do not hold the largest values.  What a row
    beside them loses is 2^-110, however small its own values."""
    gen = torch.Generator().manual_seed(7)
    big = torch.finfo(torch.bfloat16).max * 0.7
    for d in (64, 128):
        q, k, v = (0.3 * _rand(gen, 1, 8, 9, d)).bfloat16(), _rand(gen, 300, 1, d), _rand(gen, 300, 1, d)
        v[241:246] = big * torch.randint(-1, 2, (5, 1, d), generator=gen)
        _check(cuda, k, v, q, room=room, window=52, extra=2.0 ** -110)
        v[:] *= 2.0 ** -60
        v[241:246] *= 2.0 ** 60
        _check(cuda, k, v, q, room=room, window=52, extra=2.0 ** -110)


@BOTH
def test_a_key_s_size_does_not_touch_the_others_scores(cuda, room):
    """Outliers among the keys: far below every other score, or out of a row's window."""
    gen = torch.Generator().manual_seed(8)
    for d in (64, 128):
        for up in (30, 60, 90):
            q, k, v = _rand(gen, 1, 8, 9, d).abs(), _rand(gen, 300, 1, d), _rand(gen, 300, 1, d)
            k[[3, 150, 260]] = -k[[3, 150, 260]].abs() * 2.0 ** up
            _check(cuda, k, v, (0.3 * q).bfloat16(), room=room)
            k = _rand(gen, 300, 1, d)
            k[241:246] *= 2.0 ** up
            _check(cuda, k, v, (0.3 * q[:, :, 5:]).bfloat16(), room=room, window=50)  # rows 296 - 299 see 247 and up
            k *= 2.0 ** -30
            k[241:246] *= 2.0 ** 30
            _check(cuda, k, v, (2.0 ** 28 * q).bfloat16(), room=room, window=52)


@BOTH
def test_scores_of_the_smallest_factors(cuda, room):
    """Queries and a scale whose product fp32 does not hold: scores of zero, masks still masks."""
    gen = torch.Generator().manual_seed(14)
    for d in (64, 128):
        q = (2.0 ** -120 * _rand(gen, 1, 8, 9, d)).bfloat16()
        _check(cuda, _rand(gen, 150, 1, d), _rand(gen, 150, 1, d), q, room=room, scale=2.0 ** -40, window=40)


@BOTH
@pytest.mark.parametrize("softcap", [40.0, 70.0, 3e3, 1e5, 1e7, 1e30])
def test_large_softcaps(cuda, room, softcap):
    gen = torch.Generator().manual_seed(9)
    for n in (3, 40, 200):
        for size in (0.05, 0.5, 3.0):
            q = (size * _rand(gen, 1, 12, 9 if n > 9 else 3, 64)).half()
            _check(cuda, _rand(gen, n, 1, 64), _rand(gen, n, 1, 64), q, room=room, softcap=softcap, scale=0.3)


@BOTH
def test_softcap_of_the_smallest_size(cuda, room):
    """Scores that a softcap of 1e-40 leaves: all the same."""
    gen = torch.Generator().manual_seed(10)
    q = _rand(gen, 1, 12, 9, 64).bfloat16()
    q[:, ::2] = 0.0
    _check(cuda, _rand(gen, 60, 1, 64), _rand(gen, 60, 1, 64), q, room=room, softcap=1e-40)


def test_tiles_beside_other_work(cuda):
    """The many-row kernel shares the GPU with other streams' kernels: warps are held up, results are not."""
    from saint_llm_b200.ops.fp4_kv import fp4_kv_attention
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(11)
    pages, table, lengths = oracle.filled([4096, 2500], hk=1, d=128, rows=64, gen=gen, device=cuda)
    table = torch.nn.functional.pad(table, (0, 16384 - table.shape[1]), value=-1)
    q = torch.randn(2, 16, 64, 128, generator=gen).to(cuda, torch.bfloat16)
    want = fp4_kv_attention(q, pages, table, lengths)
    x = torch.randn(1 << 24, generator=gen).to(cuda)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 4]):
            if i % 4 < 2:
                x * 1.5
            else:
                outs.append(fp4_kv_attention(q, pages, table, lengths))
    torch.cuda.synchronize()
    check_errors(cuda)
    assert all(torch.equal(o, want) for o in outs)


@BOTH
@pytest.mark.parametrize("low,high", [(-126, 70), (-120, 120), (60, 124)])
def test_every_window_of_exponents(cuda, room, low, high):
    """V rows of all sizes in one tile, and queries that pick among them; beside values of 2^79 and up
    the smallest outputs lose 2^-110."""
    gen = torch.Generator().manual_seed(15)
    for d in (64, 128):
        v = _rand(gen, 260, 1, d) * 2.0 ** torch.randint(low, high + 1, (260, d // 32), generator=gen) \
            .repeat_interleave(32, -1).view(260, 1, d)
        q = (8.0 * _rand(gen, 1, 8, 9, d)).bfloat16()
        _check(cuda, _rand(gen, 260, 1, d), v, q, room=room, window=130, extra=2.0 ** -110 if high > 78 else 0.0)
