"""The 4-bit cache as a server uses it: rooms, forks and compaction keep every sequence's rows, and
beam search on it scores what a prefill of the same tokens scores."""

import pytest
import torch

from saint_llm_b200.infer.fp4_cache import Fp4KVCache, _last_logits, fp4_beam_search
from saint_llm_b200.infer.paged_kv import PoolExhausted
from saint_llm_b200.ops.pages import reserve_rows


def _model(device="cpu", dtype=torch.float32):
    from saint_llm_b200.config import ModelConfig
    from saint_llm_b200.models import SaintLLM

    cfg = ModelConfig.tiny()
    cfg = cfg.model_copy(update={"n_layers": 2, "first_dense_swa_layers": 2})
    torch.manual_seed(0)
    return SaintLLM(cfg).to(device, dtype).eval()


def _check_rows(cache, rows):
    """Every sequence reads back what was written for it (values that 4 bits hold exactly)."""
    for s, want in rows.items():
        for layer in range(cache.pool.shape[1]):
            k, v = cache.read(layer, s, len(want), dtype=torch.float32)
            assert torch.equal(k[:, 0].cpu(), want + layer) and torch.equal(v[:, 0].cpu(), -want)
    held = cache.table[cache.table >= 0].long()
    assert torch.equal(torch.bincount(held, minlength=len(cache.refcount)).int(), cache.refcount)


def _append(cache, rows, seqs, count, gen):
    dev = cache.pool.device
    new = torch.randint(0, 3, (len(seqs), count, 1), generator=gen).expand(-1, -1, 32).float()
    slots = cache.reserve(seqs, count)
    for layer in range(cache.pool.shape[1]):
        cache.write(layer, (new + layer).to(dev), -new.to(dev), slots)
    for i, s in enumerate(seqs):
        rows[s] = torch.cat([rows[s], new[i]])


def _churn(device):
    gen = torch.Generator().manual_seed(4)
    cache = Fp4KVCache(2, 40, max_seqs=5, max_len=100, head_dim=32, page_rows=16, device=device)
    rows = {s: torch.zeros(0, 32) for s in range(5)}
    _append(cache, rows, [0, 3], 20, gen)
    _append(cache, rows, [3], 13, gen)          # 33 rows
    _append(cache, rows, [0, 3, 1], 1, gen)
    cache.fork([3, 3], [2, 4])                  # part-filled last pages: copies
    rows[2], rows[4] = rows[3], rows[3]
    _check_rows(cache, rows)
    _append(cache, rows, [2, 3, 4], 5, gen)     # each its own way
    _check_rows(cache, rows)
    cache.fork([4, 2, 0], [0, 4, 3])            # all at once, sources overwritten
    rows[0], rows[4], rows[3] = rows[4], rows[2], rows[0]
    cache.free([2])
    rows[2] = rows[2][:0]
    _check_rows(cache, rows)
    used = int(cache.compact())
    assert used == int((cache.refcount > 0).sum()) and not cache.refcount[used:].any()
    _check_rows(cache, rows)
    _append(cache, rows, [2, 0, 1], 17, gen)
    _check_rows(cache, rows)
    assert cache.lengths.tolist() == [len(rows[s]) for s in range(5)]
    cache.free(range(5))
    assert not cache.refcount.any() and not cache.lengths.any()


def test_sequences_keep_their_rows():
    _churn("cpu")


@pytest.mark.gpu
def test_sequences_keep_their_rows_gpu(cuda):
    from saint_llm_b200.ops.gemm import check_errors

    _churn(cuda)
    check_errors(cuda)


def test_reserve_is_all_or_nothing():
    table, lengths = torch.full((3, 2), -1, dtype=torch.int32), torch.tensor([4, 0, 3], dtype=torch.int32)
    table[0, 0], table[2, 0] = 1, 0
    refs = torch.tensor([1, 1, 0], dtype=torch.int32)
    before = table.clone()
    with pytest.raises(PoolExhausted):
        reserve_rows(table, lengths, refs, torch.tensor([0, 1], dtype=torch.int32), 1, page_rows=4)
    with pytest.raises(IndexError):
        reserve_rows(table, lengths, refs, torch.tensor([0], dtype=torch.int32), 5, page_rows=4)
    with pytest.raises(IndexError):
        reserve_rows(table, lengths, refs, torch.tensor([3], dtype=torch.int32), 1, page_rows=4)
    assert torch.equal(table, before) and lengths.tolist() == [4, 0, 3] and refs.tolist() == [1, 1, 0]
    slots = reserve_rows(table, lengths, refs, torch.tensor([2, 0], dtype=torch.int32), 1, page_rows=4)
    assert slots.tolist() == [[3], [8]] and lengths.tolist() == [5, 0, 4] and refs.tolist() == [1, 1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("n,count,rows", [(1, 1, 16), (5, 37, 16), (1500, 3, 4), (64, 1, 64)])
def test_reserve_equals_the_definition(cuda, n, count, rows):
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 3 * rows, (n + 3,), generator=gen).int()
    width = 3 + -(-count // rows)
    pages = 5 * (n + 3) * width
    table = torch.full((n + 3, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    order = iter(torch.randperm(pages, generator=gen).tolist())
    for s, m in enumerate(lengths.tolist()):
        for c in range(-(-m // rows)):
            table[s, c] = next(order)
            refs[table[s, c]] = 1
    seqs = torch.randperm(n + 3, generator=gen)[:n].int()
    mine = [x.to(cuda) for x in (table, lengths, refs)]
    got = reserve_rows(*mine, seqs.to(cuda), count, page_rows=rows)
    want = reserve_rows(table, lengths, refs, seqs, count, page_rows=rows)
    check_errors(cuda)
    assert torch.equal(got.cpu(), want)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(mine, (table, lengths, refs), strict=True))
    # no room: nothing changes, the slots say so
    refs.fill_(1)
    full = refs.to(cuda)
    before = [x.clone() for x in mine[:2]]
    slots = reserve_rows(mine[0], mine[1], full, seqs.to(cuda), rows, page_rows=rows)
    with pytest.raises(RuntimeError, match="no free page|out of bounds"):
        check_errors(cuda)
    assert bool((slots == -1).all()) and all(torch.equal(a, b) for a, b in zip(mine[:2], before, strict=True))


def _rescore(model, ids, start):
    """Sum of log p(ids[i] | ids[:i]) for i >= start, each prefix prefilled anew in one chunk."""
    total = 0.0
    for i in range(start, ids.shape[1]):
        cache = Fp4KVCache(2, 8, max_seqs=1, max_len=64, head_dim=32, page_rows=16, device=ids.device)
        seq = torch.zeros(1, dtype=torch.int32, device=ids.device)
        total += float(torch.log_softmax(_last_logits(model, cache, ids[:, :i], seq, 0), -1)[0, ids[0, i]])
    return total


def test_beam_search_scores_what_a_prefill_scores():
    model = _model()
    prompt = torch.randint(0, 400, (2, 14), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        ids, scores = fp4_beam_search(model, prompt, beams=3, max_new_tokens=6, prefill_chunk=5, page_rows=16)
        assert ids.shape == (2, 3, 20) and bool((ids[:, :, :14] == prompt.unsqueeze(1)).all())
        assert bool((scores[:, :-1] >= scores[:, 1:]).all()) and len({tuple(x) for x in ids[0].tolist()}) == 3
        for b in range(2):
            for k in range(3):
                assert abs(_rescore(model, ids[b, k:k + 1], 14) - float(scores[b, k])) < 1e-3
        greedy, _ = fp4_beam_search(model, prompt, beams=1, max_new_tokens=6, page_rows=16)
        assert float(scores[0, 0]) >= _rescore(model, greedy[0], 14) - 1e-3


def test_beam_search_returns_a_shared_cache_empty():
    model = _model()
    cache = Fp4KVCache(2, 60, max_seqs=4, max_len=40, head_dim=32, page_rows=16)
    prompt = torch.randint(0, 400, (1, 9), generator=torch.Generator().manual_seed(2))
    a, _ = fp4_beam_search(model, prompt, beams=4, max_new_tokens=9, cache=cache)
    assert not cache.refcount.any() and (cache.table == -1).all()
    b, _ = fp4_beam_search(model, prompt, beams=4, max_new_tokens=9, cache=cache)
    assert torch.equal(a, b)


def test_refusals():
    with pytest.raises(ValueError):
        Fp4KVCache(1, 0, max_seqs=1, max_len=4)
    with pytest.raises(ValueError):
        Fp4KVCache(1, 1, max_seqs=1, max_len=4, head_dim=48)
    with pytest.raises(ValueError):
        fp4_beam_search(_model(), torch.zeros(1, 3, dtype=torch.long), beams=0, max_new_tokens=2)
    from saint_llm_b200.config import ModelConfig
    from saint_llm_b200.models import SaintLLM

    with pytest.raises(ValueError):
        fp4_beam_search(SaintLLM(ModelConfig.tiny()), torch.zeros(1, 3, dtype=torch.long), beams=2, max_new_tokens=2)
    table = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        reserve_rows(table, table[0], table[0], table[0], 0, page_rows=4)


@pytest.mark.gpu
def test_beam_search_gpu(cuda):
    from saint_llm_b200.ops.gemm import check_errors

    model = _model(cuda, torch.bfloat16)
    prompt = torch.randint(0, 400, (2, 14), generator=torch.Generator().manual_seed(1)).to(cuda)
    with torch.no_grad():
        ids, scores = fp4_beam_search(model, prompt, beams=3, max_new_tokens=6, prefill_chunk=5, page_rows=16)
        check_errors(cuda)
        # bf16 activations: a log-probability repeats to some 2^-8 of the logits' size (below 8) per token
        for k in range(3):
            assert abs(_rescore(model, ids[0, k:k + 1], 14) - float(scores[0, k])) < 6 * 8 * 2.0 ** -7
        check_errors(cuda)


@pytest.mark.gpu
def test_decode_step_in_a_cuda_graph(cuda):
    """Reserve, write and attention of one step, captured once and replayed across page boundaries."""
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(3)
    make = lambda: Fp4KVCache(1, 30, max_seqs=3, max_len=64, head_dim=64, page_rows=16, device=cuda)  # noqa: E731
    a, b = make(), make()
    seqs = torch.arange(3, dtype=torch.int32, device=cuda)
    k, v = torch.zeros(3, 1, 64, device=cuda, dtype=torch.bfloat16), torch.zeros(3, 1, 64, device=cuda, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 1, 64, device=cuda, dtype=torch.bfloat16)

    def step(cache):
        cache.write(0, k, v, cache.reserve(seqs, 1))
        return cache.attend(0, q)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm-up on another cache
        step(make())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    for _ in range(40):
        k.copy_(torch.randn(3, 1, 64, generator=gen))
        v.copy_(torch.randn(3, 1, 64, generator=gen))
        q.copy_(torch.randn(3, 4, 1, 64, generator=gen))
        graph.replay()
        assert torch.equal(out, step(b))
    assert torch.equal(a.table, b.table) and a.lengths.tolist() == [40, 40, 40]
    check_errors(cuda)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_state_keeps_its_addresses(device, request):
    if device == "cuda":
        request.getfixturevalue("cuda")
    cache = Fp4KVCache(1, 8, max_seqs=3, max_len=64, head_dim=32, page_rows=16, device=device)
    state = [cache.table, cache.lengths, cache.refcount]
    where = [t.data_ptr() for t in state]
    cache.reserve([1], 40)
    cache.fork([1], [0])
    cache.free([1])
    cache.compact()
    assert [t.data_ptr() for t in (cache.table, cache.lengths, cache.refcount)] == where
    assert state[0].tolist() == [[0, 1, 2, -1], [-1] * 4, [-1] * 4] and state[1].tolist() == [40, 0, 0]
    assert state[2].tolist() == [1, 1, 1, 0, 0, 0, 0, 0]


@pytest.mark.gpu
def test_captured_step_follows_forks_and_compaction(cuda):
    from saint_llm_b200.ops.gemm import check_errors

    gen = torch.Generator().manual_seed(8)
    make = lambda: Fp4KVCache(1, 30, max_seqs=3, max_len=96, head_dim=64, page_rows=16, device=cuda)  # noqa: E731
    a, b = make(), make()
    seqs = torch.arange(3, dtype=torch.int32, device=cuda)
    k, v = (torch.zeros(3, 1, 64, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    q = torch.zeros(3, 4, 1, 64, device=cuda, dtype=torch.bfloat16)

    def step(cache):
        cache.write(0, k, v, cache.reserve(seqs, 1))
        return cache.attend(0, q)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm-up on another cache
        step(make())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    for i in range(24):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=gen))
        graph.replay()
        assert torch.equal(out, step(b))
        for cache in (a, b):
            if i % 5 == 2:
                cache.fork([2, 0], [0, 1])
            if i % 7 == 3:
                cache.compact()
    assert torch.equal(a.table, b.table) and torch.equal(a.refcount, b.refcount)
    check_errors(cuda)


def test_sequences_out_of_range_are_refused():
    cache = Fp4KVCache(1, 4, max_seqs=2, max_len=32, head_dim=32, page_rows=16)
    cache.reserve([0, 1], 3)
    q = torch.zeros(1, 2, 1, 32, dtype=torch.bfloat16)
    for seqs in ([2], [-1], torch.tensor([5])):
        with pytest.raises(IndexError):
            cache.attend(0, q, seqs)
    for seq, length in ((2, 1), (-1, 1), (0, 33), (0, -1)):
        with pytest.raises(IndexError):
            cache.read(0, seq, length)


@pytest.mark.gpu
def test_sequences_out_of_range_are_recorded(cuda):
    from saint_llm_b200.ops.gemm import check_errors

    cache = Fp4KVCache(1, 4, max_seqs=2, max_len=32, head_dim=32, page_rows=16, device=cuda)
    gen = torch.Generator().manual_seed(2)
    k = torch.randn(2, 3, 32, generator=gen).to(cuda)
    cache.write(0, k, k, cache.reserve([0, 1], 3))
    q = torch.randn(2, 4, 1, 32, generator=gen).to(cuda, torch.bfloat16)
    good = cache.attend(0, q, [0, 1])
    check_errors(cuda)
    for wrong in (2, -1):
        out = cache.attend(0, q, torch.tensor([0, wrong], device=cuda))
        assert torch.equal(out[0], good[0])
        with pytest.raises(RuntimeError, match="out of bounds"):
            check_errors(cuda)
    with pytest.raises(IndexError):
        cache.read(0, 0, 33)
    check_errors(cuda)
