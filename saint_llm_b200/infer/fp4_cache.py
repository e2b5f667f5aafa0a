"""A K / V cache of many sequences and layers in 4-bit pages, and beam search on it.

``Fp4KVCache`` owns one pool (a page holds ``page_rows`` tokens of every layer), a block table,
lengths and reference counts, all on the device:

* ``reserve`` opens room for the next tokens of some sequences and returns their slots;
* ``write`` quantises a layer's K / V rows into the slots, ``attend`` reads them where they lie,
  ``read`` returns them in bf16;
* ``fork`` makes sequences copies of others (pages shared, part-filled last pages copied), ``free``
  ends them, ``compact`` moves the pages in use to the front of the pool.

At 4.25 bits a value a page takes 0.27 of its bf16 size.  Nothing is read on the host and the state
keeps its addresses, so a step captured in a CUDA graph follows forks and compactions between its
replays; what went wrong on the device -- no free page, an index out of range -- is raised by
``ops.gemm.check_errors``.

Lengths grow by ``reserve`` and are replaced by ``fork`` and ``free``: single tokens are not taken back
(a smaller number written into ``lengths`` would leave their pages behind), and pages that lie
behind every window are kept.

``fp4_beam_search`` decodes sliding-window models with it: one prefill per prompt, a fork to all
beams, then a reserve, one write and attention per layer, and a fork per step.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor, nn

from saint_llm_b200.models.attention import SWAttention
from saint_llm_b200.models.attention.common import rope_tables
from saint_llm_b200.models.mhc import MHC
from saint_llm_b200.ops import pages as page_ops
from saint_llm_b200.ops.fp4_kv import fp4_kv_attention, fp4_kv_read, fp4_kv_slab_bytes, fp4_kv_write
from saint_llm_b200.ops.gemm import check_errors


class Fp4KVCache:
    def __init__(self, n_layers: int, n_pages: int, *, max_seqs: int, max_len: int, kv_heads: int = 1,
                 head_dim: int = 128, page_rows: int = 64, device: torch.device | str | None = None) -> None:
        if min(n_layers, n_pages, max_seqs, max_len, kv_heads) <= 0:
            raise ValueError("layers, pages, sequences, length and heads must be positive")
        self.page_rows, self.head_dim, self.max_len = page_rows, head_dim, max_len
        slab = fp4_kv_slab_bytes(page_rows, head_dim)
        self.pool = torch.zeros(n_pages, n_layers, kv_heads, slab, dtype=torch.uint8, device=device)
        ints = {"dtype": torch.int32, "device": device}
        self.table = torch.full((max_seqs, -(-max_len // page_rows)), -1, **ints)
        self.lengths = torch.zeros(max_seqs, **ints)
        self.refcount = torch.zeros(n_pages, **ints)

    def nbytes(self) -> int:
        return self.pool.numel()

    def _ids(self, seqs: Tensor | Sequence[int]) -> Tensor:
        if isinstance(seqs, Tensor):
            return seqs.to(device=self.table.device, dtype=torch.int32)
        return torch.tensor(list(seqs), dtype=torch.int32, device=self.table.device)

    def reserve(self, seqs: Tensor | Sequence[int], count: int) -> Tensor:
        """Slots (n, count) int64 of the next ``count`` tokens of sequences ``seqs``."""
        return page_ops.reserve_rows(self.table, self.lengths, self.refcount, self._ids(seqs), count,
                                     page_rows=self.page_rows)

    def write(self, layer: int, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """K / V rows (n, count, head_dim) or (n, count, kv_heads, head_dim) of a layer into ``slots``."""
        shape = (slots.numel(), self.pool.shape[2], self.head_dim)
        fp4_kv_write(k.reshape(shape), v.reshape(shape), self.pool[:, layer], slots.reshape(-1))

    def read(self, layer: int, seq: int, length: int, *, dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
        """The first ``length`` K and V rows (length, kv_heads, head_dim) of a sequence."""
        if not 0 <= seq < self.table.shape[0] or not 0 <= length <= self.table.shape[1] * self.page_rows:
            raise IndexError(f"{length} rows of sequence {seq}: the cache has {self.table.shape[0]} sequences of up to "
                             f"{self.table.shape[1] * self.page_rows}")
        pos = torch.arange(length, device=self.table.device)
        slots = self.table[seq, pos // self.page_rows].long() * self.page_rows + pos % self.page_rows
        return fp4_kv_read(self.pool[:, layer], slots, head_dim=self.head_dim, dtype=dtype)

    def attend(self, layer: int, q: Tensor, seqs: Tensor | Sequence[int] | None = None, *, window: int = 0,
               sink: Tensor | None = None, softcap: float | None = None) -> Tensor:
        """Attention of the last T tokens, q (n, H, T, head_dim), of ``seqs`` (default: all of them)."""
        table, lengths = self.table, self.lengths
        if seqs is not None:
            ids = self._ids(seqs).long()
            at = ids.clamp(0, table.shape[0] - 1)
            if not ids.is_cuda and not torch.equal(ids, at):
                raise IndexError(f"sequences {ids.tolist()} of {table.shape[0]}")
            # on CUDA a length that no table holds records the error where the kernel reads it
            table, lengths = table[at], torch.where(ids == at, lengths[at], torch.iinfo(torch.int32).max)
        return fp4_kv_attention(q, self.pool[:, layer], table, lengths, window=window, sink=sink, softcap=softcap)

    def fork(self, parents: Tensor | Sequence[int], children: Tensor | Sequence[int]) -> None:
        """Sequences ``children`` become copies of ``parents`` as they are now (-1: empty)."""
        state = page_ops.fork_pages(self.pool, self.table, self.lengths, self.refcount, self._ids(parents),
                                    self._ids(children), page_rows=self.page_rows)
        for mine, new in zip((self.table, self.lengths, self.refcount), state, strict=True):
            mine.copy_(new)

    def free(self, seqs: Tensor | Sequence[int]) -> None:
        ids = self._ids(seqs)
        self.fork(torch.full_like(ids, -1), ids)

    def compact(self) -> Tensor:
        """Pages in use to the front of the pool; returns how many there are (device scalar)."""
        table, refcount, used = page_ops.compact_pages(self.pool, self.table, self.refcount)
        self.table.copy_(table)
        self.refcount.copy_(refcount)
        return used


def _check_model(model: nn.Module) -> None:
    for blk in model.blocks:  # type: ignore[attr-defined]
        if type(blk.attention) is not SWAttention:
            raise ValueError("the 4-bit cache decodes models of sliding-window layers")
    if model.cfg.n_sink_tokens:  # type: ignore[attr-defined]
        raise ValueError("the 4-bit cache does not support prepended sink tokens")


def _check_cache(model: nn.Module, cache: Fp4KVCache, n: int, length: int, device: torch.device) -> None:
    d = model.cfg.attention.head_dim  # type: ignore[attr-defined]
    if cache.pool.shape[1] < len(model.blocks) or cache.pool.shape[2] != 1 or cache.head_dim != d:  # type: ignore[attr-defined]
        raise ValueError(f"the cache holds {cache.pool.shape[1]} layers of {cache.pool.shape[2]} heads of {cache.head_dim}, the "
                         f"model has {len(model.blocks)} of 1 head of {d}")  # type: ignore[attr-defined]
    if cache.pool.device != device:
        raise ValueError(f"the cache is on {cache.pool.device}, the prompts are on {device}")
    if n > cache.table.shape[0] or length > cache.table.shape[1] * cache.page_rows:
        raise ValueError(f"{n} sequences of {length} rows: the cache has {cache.table.shape[0]} sequences of up to "
                         f"{cache.table.shape[1] * cache.page_rows}")
    if bool(cache.lengths[:n].any()):
        raise ValueError(f"sequences 0 .. {n - 1} of the cache must be empty")


def _last_logits(model: nn.Module, cache: Fp4KVCache, ids: Tensor, seqs: Tensor, start: int) -> Tensor:
    """(n, V) logits after the tokens ``ids`` (n, T) of sequences ``seqs``, which stand at ``start``."""
    cfg = model.cfg  # type: ignore[attr-defined]
    slots = cache.reserve(seqs, ids.shape[1])
    cos, sin = rope_tables(ids.shape[1], cfg.attention.rope_dim, cfg.attention.rope_theta, ids.device, start=start)
    x = MHC.expand(model._embed_inputs(ids, None, None), cfg.mhc.expansion_factor)  # type: ignore[attr-defined]
    vis = ids == cfg.tokenizer_slots.image_pad
    for layer, blk in enumerate(model.blocks):  # type: ignore[attr-defined]
        a = blk.attention
        inner, _, b_l, c_l = blk.attn_mhc.split(x)
        q = a._queries(inner, cos, sin)
        cache.write(layer, *a._sw_kv(inner, cos, sin), slots)
        if q.is_cuda and q.dtype == torch.float32:
            q = q.bfloat16()  # the kernels take 16 bits; bf16 keeps fp32's range, for outputs as large as V is
        out = cache.attend(layer, q, seqs, window=a.attn_cfg.sliding_window_size, sink=a.sink_logit,
                           softcap=a.attn_cfg.logit_softcap)
        x = blk.attn_mhc.combine(x, a.output(out.to(x.dtype)), b_l, c_l)
        inner, _, b_l, c_l = blk.moe_mhc.split(x)
        x = blk.moe_mhc.combine(x, blk.moe(inner, token_ids=ids, is_visual=vis), b_l, c_l)
        if blk.side_channel.active:
            collapsed = x.mean(-2)
            x = x + ((blk.side_channel(collapsed) - collapsed) / x.shape[-2]).unsqueeze(-2)
    h = model.final_norm(MHC.collapse(x))  # type: ignore[attr-defined]
    return model.logits(h[:, -1:]).squeeze(1).float()  # type: ignore[attr-defined]


@torch.no_grad()
def fp4_beam_search(model: nn.Module, prompt_ids: Tensor, *, beams: int, max_new_tokens: int,
                    prefill_chunk: int = 256, page_rows: int = 64,
                    cache: Fp4KVCache | None = None) -> tuple[Tensor, Tensor]:
    """Beam search of prompts (B, T) on a 4-bit cache: the ids (B, beams, T + max_new_tokens) and the
    sums of log-probabilities (B, beams), best first.  Prompts are prefilled once, in chunks; the
    beams of a prompt share its pages.  ``cache`` (its sequences 0 .. B * beams - 1 empty) is used
    and emptied again, whatever happens; by default one of the size needed is made.  A cache that
    does not fit the model or the request is refused; one whose pool runs out of pages raises
    ``PoolExhausted`` (on CUDA ``RuntimeError``, after the last step).  On CUDA the attention of an
    fp32 model takes its queries and gives its outputs in bf16."""
    _check_model(model)
    b, t = prompt_ids.shape
    n = b * beams
    if beams <= 0 or max_new_tokens <= 0 or t == 0 or prefill_chunk <= 0:
        raise ValueError("beams, max_new_tokens, prefill_chunk and the prompt's length must be positive")
    cfg, dev = model.cfg, prompt_ids.device  # type: ignore[attr-defined]
    if beams > cfg.vocab_size:
        raise ValueError(f"{beams} beams of {cfg.vocab_size} tokens")
    total = t + max_new_tokens
    if cache is None:
        # the prompts, and for every beam its own pages from the prompt's last one on, twice during a fork
        own = -(-total // page_rows) - t // page_rows + 1
        cache = Fp4KVCache(len(model.blocks), b * (-(-t // page_rows)) + 2 * n * own, max_seqs=n,  # type: ignore[attr-defined]
                           max_len=total, head_dim=cfg.attention.head_dim, page_rows=page_rows, device=dev)
    else:
        _check_cache(model, cache, n, total - 1, dev)  # the last tokens are not fed
    every = torch.arange(n, dtype=torch.int32, device=dev)
    first = every[::beams].contiguous()
    try:
        logits = None
        for c in range(0, t, prefill_chunk):
            logits = _last_logits(model, cache, prompt_ids[:, c:c + prefill_chunk], first, c)
        cache.fork(first.repeat_interleave(beams), every)
        logp = torch.log_softmax(logits, -1)
        scores, tokens = logp.topk(beams, -1)  # (B, beams)
        ids = torch.cat([prompt_ids.repeat_interleave(beams, 0), tokens.reshape(n, 1)], 1)
        for step in range(1, max_new_tokens):
            logp = torch.log_softmax(_last_logits(model, cache, ids[:, -1:], every, t + step - 1), -1)
            scores, pick = (scores.unsqueeze(-1) + logp.view(b, beams, -1)).flatten(1).topk(beams, -1)
            parents = (pick // logp.shape[-1] + torch.arange(b, device=dev).unsqueeze(1) * beams).reshape(-1)
            ids = torch.cat([ids[parents], (pick % logp.shape[-1]).reshape(n, 1)], 1)
            if step + 1 < max_new_tokens:  # the last tokens are not fed again
                cache.fork(parents, every)
    finally:
        cache.free(every)
    if dev.type == "cuda":
        check_errors(dev)  # no free page, an index out of range: the tokens would be made without some rows
    return ids.view(b, beams, -1), scores


__all__ = ["Fp4KVCache", "fp4_beam_search"]
