"""Beam search on the 4-bit cache against the model itself: with the cache's rows kept in fp32, what it
scores is what the model scores; a step's fork matters; a cache that does not fit is refused."""

import math

import pytest
import torch

from saint_llm_b200.infer.fp4_cache import Fp4KVCache, _last_logits, fp4_beam_search
from saint_llm_b200.infer.paged_kv import PoolExhausted


class ExactCache(Fp4KVCache):
    """Rows in fp32 beside the pages (which still are what forks copy: a page's rows follow its bytes here too)."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        pages, layers = self.pool.shape[:2]
        self.pool = torch.zeros(pages, layers, 1, 2, self.page_rows, self.head_dim)

    def write(self, layer, k, v, slots):
        page, row = slots.reshape(-1) // self.page_rows, slots.reshape(-1) % self.page_rows
        self.pool[page, layer, 0, 0, row] = k.reshape(-1, self.head_dim)
        self.pool[page, layer, 0, 1, row] = v.reshape(-1, self.head_dim)

    def attend(self, layer, q, seqs=None, *, window=0, sink=None, softcap=None):
        ids = range(len(q)) if seqs is None else seqs.tolist()
        out = torch.zeros_like(q, dtype=torch.float64)
        for i, s in enumerate(ids):
            n = int(self.lengths[s])
            k, v = (self.pool[self.table[s].clamp(min=0), layer, 0, x].reshape(-1, self.head_dim)[:n].double() for x in (0, 1))
            for t in range(q.shape[2]):
                at = n - q.shape[2] + t
                lo = max(0, at - window + 1) if window else 0
                score = q[i, :, t].double() @ k[lo:at + 1].T / math.sqrt(self.head_dim)
                if softcap:
                    score = softcap * torch.tanh(score / softcap)
                p = score.exp()
                total = p.sum(-1, keepdim=True)
                if sink is not None:
                    total = total + sink.double().exp().unsqueeze(-1)
                out[i, :, t] = p @ v[lo:at + 1] / total
        return out


def _model(device="cpu", dtype=torch.float32):
    """Two sliding-window layers (window 8) and a head of its own, random: beams differ, and change places."""
    from saint_llm_b200.config import ModelConfig
    from saint_llm_b200.models import SaintLLM

    cfg = ModelConfig.tiny().model_copy(update={"n_layers": 2, "first_dense_swa_layers": 2,
                                                        "tie_word_embeddings": False})
    torch.manual_seed(0)
    model = SaintLLM(cfg)
    gen = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if p.dim() >= 2:
                p.copy_(torch.randn(p.shape, generator=gen) * (0.3 if "embed" in name else p.shape[-1] ** -0.5))
            if "sink" in name:
                p.copy_(torch.randn(p.shape, generator=gen))
    return model.to(device, dtype).eval()


def _exact(n, *, pages=60, length=64):
    return ExactCache(2, pages, max_seqs=n, max_len=length, head_dim=32, page_rows=16)


def _prompt(b, t, seed=1):
    return torch.randint(0, 400, (b, t), generator=torch.Generator().manual_seed(seed))


def test_a_prefill_in_chunks_gives_the_model_s_logits():
    model, ids = _model(), _prompt(2, 37)
    with torch.no_grad():
        for chunk in (37, 11, 1):
            cache, seqs = _exact(2), torch.arange(2, dtype=torch.int32)
            for c in range(0, 37, chunk):
                got = _last_logits(model, cache, ids[:, c:c + chunk], seqs, c)
                want = model(ids[:, :c + chunk])["logits"][:, -1]
                assert want.std() > 0.1 and torch.allclose(got, want, rtol=1e-4, atol=1e-4)


def _scores_of_the_model(model, ids, start):
    logp = torch.log_softmax(model(ids)["logits"].float(), -1)[:, start - 1:-1]
    return logp.gather(-1, ids[:, start:].unsqueeze(-1)).sum((1, 2))


class Forks:
    """The forks of a search, and whether one after the first moved a beam's rows to one with other tokens."""

    def __init__(self, cache, skip=False):
        self.calls, self.fork, self.skip = [], cache.fork, skip
        cache.fork = self

    def __call__(self, parents, children):
        self.calls.append(torch.as_tensor(parents).tolist())
        if not self.skip or len(self.calls) == 1 or min(self.calls[-1]) < 0:
            self.fork(parents, children)


def test_beams_that_change_places_keep_their_rows():
    model, prompt = _model(), _prompt(2, 13)
    with torch.no_grad():
        cache = _exact(8)
        forks = Forks(cache)
        ids, scores = fp4_beam_search(model, prompt, beams=4, max_new_tokens=9, prefill_chunk=5, cache=cache)
        moves = [c for c in forks.calls[1:-1] if c != list(range(8))]
        assert moves and len({tuple(x) for x in ids[0, :, 13:20].tolist()}) > 1
        want = _scores_of_the_model(model, ids.flatten(0, 1), 13).view(2, 4)
        assert torch.allclose(scores, want, rtol=0, atol=1e-3)
        # without the forks of its steps a search scores other rows than its beams'
        cache = _exact(8)
        Forks(cache, skip=True)
        ids, scores = fp4_beam_search(model, prompt, beams=4, max_new_tokens=9, prefill_chunk=5, cache=cache)
        want = _scores_of_the_model(model, ids.flatten(0, 1), 13).view(2, 4)
        assert float((scores - want).abs().max()) > 0.1


def test_four_bits_score_near_the_model():
    """K and V lose a few per cent to their 4 bits; a wrong window, order or position loses far more."""
    model, ids = _model(), _prompt(2, 30)
    with torch.no_grad():
        cache = Fp4KVCache(2, 8, max_seqs=2, max_len=64, head_dim=32, page_rows=16)
        got = _last_logits(model, cache, ids, torch.arange(2, dtype=torch.int32), 0)
        want = model(ids)["logits"][:, -1]
    assert float((got - want).norm() / want.norm()) < 0.25


def test_a_cache_that_does_not_fit_is_refused():
    model, prompt = _model(), _prompt(1, 9)
    search = lambda **kw: fp4_beam_search(model, prompt, beams=4, max_new_tokens=9, **kw)  # noqa: E731
    kw = {"max_seqs": 4, "max_len": 40, "head_dim": 32, "page_rows": 16}
    for wrong in (Fp4KVCache(1, 60, **kw), Fp4KVCache(2, 60, **{**kw, "max_seqs": 3}), Fp4KVCache(2, 60, **{**kw, "max_len": 16}),
                  Fp4KVCache(2, 60, **{**kw, "head_dim": 64}), Fp4KVCache(2, 60, kv_heads=2, **kw)):
        with pytest.raises(ValueError):
            search(cache=wrong)
        assert not wrong.refcount.any()
    used = Fp4KVCache(2, 60, **kw)
    used.reserve([2], 3)
    with pytest.raises(ValueError, match="empty"):
        search(cache=used)
    with pytest.raises(ValueError):
        fp4_beam_search(model, prompt, beams=10 ** 6, max_new_tokens=2)
    with pytest.raises(ValueError):
        fp4_beam_search(model, prompt, beams=2, max_new_tokens=2, prefill_chunk=0)
    ok = Fp4KVCache(2, 60, **{**kw, "max_len": 17})  # the last token is never fed: 17 rows
    search(cache=ok)


def test_a_search_that_fails_leaves_the_cache_empty():
    model, prompt = _model(), _prompt(1, 9)
    cache = Fp4KVCache(2, 3, max_seqs=4, max_len=40, head_dim=32, page_rows=16)
    with pytest.raises(PoolExhausted):
        fp4_beam_search(model, prompt, beams=4, max_new_tokens=9, cache=cache)
    assert not cache.refcount.any() and not cache.lengths.any() and bool((cache.table == -1).all())


@pytest.mark.gpu
def test_a_search_without_pages_raises_on_the_gpu(cuda):
    from saint_llm_b200.ops.gemm import check_errors

    model, prompt = _model(cuda, torch.bfloat16), _prompt(1, 9).to(cuda)
    cache = Fp4KVCache(2, 3, max_seqs=4, max_len=40, head_dim=32, page_rows=16, device=cuda)
    with pytest.raises(RuntimeError, match="no free page"):
        fp4_beam_search(model, prompt, beams=4, max_new_tokens=9, cache=cache)
    check_errors(cuda)
    assert not cache.refcount.any() and not cache.lengths.any() and bool((cache.table == -1).all())


@pytest.mark.gpu
def test_four_bits_on_the_gpu_score_near_the_cpu(cuda):
    """The same model and tokens; bf16 activations and products in another order."""
    model, ids = _model(), _prompt(2, 30)
    want = {}
    for device, dtype in (("cpu", torch.float32), (cuda, torch.float32), (cuda, torch.bfloat16)):
        cache = Fp4KVCache(2, 8, max_seqs=2, max_len=64, head_dim=32, page_rows=16, device=device)
        mine = model.to(device, dtype)
        with torch.no_grad():
            got = _last_logits(mine, cache, ids.to(device), torch.arange(2, dtype=torch.int32, device=device), 0)
        want[(str(device), dtype)] = got.float().cpu()
    first, *others = want.values()
    for got in others:
        assert float((got - first).norm() / first.norm()) < 0.25
