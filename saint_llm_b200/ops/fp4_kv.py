"""A paged K / V cache held in 4 bits: write, read and attention on the pages.

Rows are MXFP4 along ``head_dim`` (the format of ``ops.quant``): E2M1 elements, one E8M0 scale
per 32, 4.25 bits per value, so a pool of given size holds 3.76 times the tokens of a bf16 one.

``pages`` is a uint8 tensor (n_pages, kv_heads, slab), ``slab = page_rows * head_dim * 17 / 16``:
the K codes (page_rows x head_dim / 2), the V codes, the K scales (page_rows x head_dim / 32) and
the V scales.  Byte j of a row's codes holds dim 2j in its low four bits and dim 2j + 1 in its
high ones.  ``page_rows`` is a multiple of 16, ``head_dim`` 32, 64 or 128.  A view of a larger
pool works too as long as each page is contiguous (``pool[:, layer]`` of a pool
(n_pages, layers, kv_heads, slab)).

Quantisation: the scale's exponent is the smallest e with amax <= 6 * 2^e (at least -126), an
element goes to the nearest level and a tie to the smaller one, a negative value that rounds to
zero becomes +0.  A block that holds a NaN or an infinity reads back as NaN.

CPU tensors (and ``backend.eager_mode()``) take the definitions below; CUDA tensors run
``csrc/fp4_kv.cu``.  An index outside the pool or the table is recorded on the device and raised
by ``ops.gemm.check_errors``; the row it names is skipped.  The definitions raise ``IndexError``.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from saint_llm_b200.ops import backend
from saint_llm_b200.ops.gemm import error_word
from saint_llm_b200.ops.quant import FP4_E2M1_LEVELS

BLOCK = 32
_ROW_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def fp4_kv_slab_bytes(page_rows: int, head_dim: int) -> int:
    """Bytes of one page of one K / V head."""
    if head_dim not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32, 64 or 128; got {head_dim}")
    if page_rows <= 0 or page_rows % 16:
        raise ValueError(f"page_rows must be a positive multiple of 16; got {page_rows}")
    return page_rows * head_dim * 17 // 16


def fp4_kv_page_rows(pages: Tensor, head_dim: int) -> int:
    """Rows per page of a pages tensor, from its slab size."""
    if pages.dim() != 3 or pages.dtype != torch.uint8:
        raise ValueError(f"pages must be uint8 (n_pages, kv_heads, slab); got {tuple(pages.shape)} {pages.dtype}")
    rows = pages.shape[2] * 16 // (17 * head_dim)
    if rows <= 0 or fp4_kv_slab_bytes(rows, head_dim) != pages.shape[2]:
        raise ValueError(f"a slab of {pages.shape[2]} bytes is no page of head_dim {head_dim}")
    return rows


def _parts(pages: Tensor, rows: int, d: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """K codes, V codes (n, heads, rows, d/2) and K scales, V scales (n, heads, rows, d/32), as views."""
    c, s = rows * d // 2, rows * d // BLOCK
    cuts = (pages[..., :c], pages[..., c:2 * c], pages[..., 2 * c:2 * c + s], pages[..., 2 * c + s:])
    return tuple(x.unflatten(-1, (rows, -1)) for x in cuts)  # type: ignore[return-value]


def _encode(x: Tensor) -> tuple[Tensor, Tensor]:
    """x (..., d) -> packed codes (..., d / 2) and scale bytes (..., d / 32)."""
    blocks = x.float().unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 3 + (m > 0.75).int(), torch.full_like(e, -126)).clamp(-126, 126)
    ok = torch.isfinite(amax)
    mag = torch.where(ok.unsqueeze(-1), blocks.abs() * ((127 - e) << 23).view(torch.float32).unsqueeze(-1), 0.0)
    levels = FP4_E2M1_LEVELS.to(x.device)
    code = torch.bucketize(mag, (levels[1:] + levels[:-1]) / 2, right=False)  # a tie goes down
    code = torch.where((blocks < 0) & (code > 0), code + 8, code).to(torch.uint8).flatten(-2)
    byte = torch.where(ok, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def _decode(codes: Tensor, scales: Tensor) -> Tensor:
    """The fp32 values (..., d) of packed codes and scale bytes."""
    levels = FP4_E2M1_LEVELS.to(codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    s = (scales.int() << 23).view(torch.float32)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (torch.cat((levels, -levels))[c].unflatten(-1, (-1, BLOCK)) * s.unsqueeze(-1)).flatten(-2)


def _check_slots(slots: Tensor, n_slots: int) -> Tensor:
    """The rows that are written or read; raises on a slot outside the pool (host check: CPU tensors)."""
    if bool(((slots < -1) | (slots >= n_slots)).any()):
        raise IndexError(f"slots must be in [-1, {n_slots})")
    return slots >= 0


def fp4_kv_write(k: Tensor, v: Tensor, pages: Tensor, slots: Tensor) -> None:
    """Quantise rows ``k``, ``v`` (N, kv_heads, head_dim; bf16, fp16 or fp32, any strides) into
    ``pages`` at ``slots`` (N,) int64 = page * page_rows + row, in place.  -1 skips a row; the
    other slots must differ from one another."""
    if backend.native_for(pages):
        backend.ext().fp4_kv_write(k, v, pages, slots, error_word(pages.device))
        return
    if k.dim() != 3 or v.shape != k.shape or v.dtype != k.dtype or k.dtype not in _ROW_TYPES:
        raise ValueError("k and v must be (rows, kv_heads, head_dim) of one type in bf16, fp16 or fp32")
    rows = fp4_kv_page_rows(pages, k.shape[2])
    if slots.dtype != torch.int64 or slots.shape != k.shape[:1] or k.shape[1] != pages.shape[1]:
        raise ValueError("slots must be int64 with one entry per row, rows of the pages' heads")
    live = _check_slots(slots, pages.shape[0] * rows)
    page, row = slots[live] // rows, slots[live] % rows
    kc, vc, ks, vs = _parts(pages, rows, k.shape[2])
    for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
        c, s = _encode(x[live])
        codes[page, :, row], scales[page, :, row] = c, s


def fp4_kv_read(pages: Tensor, slots: Tensor, *, head_dim: int,
                dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
    """The K and V rows (N, kv_heads, head_dim) at ``slots`` (N,) int64 in ``dtype``; -1 gives zeros."""
    if backend.native_for(pages):
        return backend.ext().fp4_kv_read(pages, slots, head_dim, dtype, error_word(pages.device))
    if dtype not in _ROW_TYPES:
        raise ValueError("rows are read in bf16, fp16 or fp32")
    rows = fp4_kv_page_rows(pages, head_dim)
    if slots.dtype != torch.int64 or slots.dim() != 1:
        raise ValueError("slots must be an int64 vector")
    live = _check_slots(slots, pages.shape[0] * rows)
    at = slots.clamp(min=0)
    kc, vc, ks, vs = (x[at // rows, :, at % rows] for x in _parts(pages, rows, head_dim))
    keep = live.view(-1, 1, 1)
    zero = torch.zeros((), device=pages.device)
    return (torch.where(keep, _decode(kc, ks), zero).to(dtype), torch.where(keep, _decode(vc, vs), zero).to(dtype))


def _check_table(pages: Tensor, table: Tensor, lengths: Tensor, rows: int, tokens: int, window: int) -> None:
    """Raises where a key that some query sees is in no page of the pool (host check: CPU tensors)."""
    room = table.shape[1] * rows
    if bool((lengths > room).any()):
        raise IndexError(f"lengths must be at most {room}, the rows of a table row's pages")
    first = (lengths - tokens + 1 - window).clamp(min=0) if window > 0 else torch.zeros_like(lengths)
    page = torch.arange(table.shape[1], device=table.device).unsqueeze(0)
    seen = (page * rows < lengths.unsqueeze(1)) & ((page + 1) * rows > first.unsqueeze(1))
    if bool((seen & ((table < 0) | (table >= pages.shape[0]))).any()):
        raise IndexError(f"table ids must be in [0, {pages.shape[0]})")


def fp4_kv_attention_reference(q: Tensor, pages: Tensor, table: Tensor, lengths: Tensor, *, window: int = 0,
                               sink: Tensor | None = None, softcap: float | None = None,
                               scale: float | None = None) -> Tensor:
    """The definition of ``fp4_kv_attention`` in the precision of ``q`` widened to at least 32 bits."""
    b, h, t, d = q.shape
    rows = fp4_kv_page_rows(pages, d)
    hk = pages.shape[1]
    wide = torch.promote_types(q.dtype, torch.float32)
    kc, vc, ks, vs = _parts(pages[table.long().clamp(0, pages.shape[0] - 1)], rows, d)  # (B, P, heads, rows, ...)
    n = table.shape[1] * rows
    k = _decode(kc, ks).transpose(1, 2).reshape(b, hk, 1, n, d).to(wide)
    v = _decode(vc, vs).transpose(1, 2).reshape(b, hk, 1, n, d).to(wide)
    key = torch.arange(n, device=q.device)
    length = lengths.view(b, 1, 1).long()
    pos = length - t + torch.arange(t, device=q.device).view(1, t, 1)
    seen = key <= pos
    if window > 0:
        seen = seen & (key > pos - window)
    live = (key < length).view(b, 1, 1, n, 1)
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)  # rows behind the length may hold anything
    s = torch.einsum("bkgtd,bkgnd->bkgtn", q.to(wide).view(b, hk, h // hk, t, d), k.expand(b, hk, h // hk, n, d))
    s = s * (1.0 / math.sqrt(d) if scale is None else scale)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = s.masked_fill(~seen.view(b, 1, 1, t, n), float("-inf"))
    m = s.amax(-1, keepdim=True)
    if sink is not None:
        m = torch.maximum(m, sink.to(wide).view(1, hk, h // hk, 1, 1))
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink.to(wide).view(1, hk, h // hk, 1, 1) - m)
    # a block that reads as NaN reaches the queries that see its key, and no others (0 times NaN would)
    bad = v.isnan()
    out = torch.einsum("bkgtn,bkgnd->bkgtd", p, torch.where(bad, 0.0, v).expand(b, hk, h // hk, n, d))
    hit = torch.einsum("btn,bknd->bktd", seen.expand(b, t, n).to(wide), bad.squeeze(2).to(wide)) > 0
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.where(hit.unsqueeze(2), float("nan"), out)
    return out.reshape(b, h, t, d).to(q.dtype)


def fp4_kv_attention(q: Tensor, pages: Tensor, table: Tensor, lengths: Tensor, *, window: int = 0,
                     sink: Tensor | None = None, softcap: float | None = None, scale: float | None = None) -> Tensor:
    """Attention of the last T tokens of each sequence over its pages.

    ``q`` (B, H, T, head_dim) or (B, H, head_dim) in bf16 or fp16, any strides; ``table`` (B, P)
    int32 block tables (-1 padded) and ``lengths`` (B,) int32 rows per sequence, the T tokens
    included (their K / V are written first).  Query t stands at position ``length - T + t`` and
    sees the keys up to it, the last ``window`` of them if ``window > 0``.  H is a multiple of the
    pages' K / V heads; query head h reads K / V head ``h // (H / kv_heads)``.  ``sink`` (H,): a
    logit that joins the denominator; ``softcap``: scores become ``c tanh(s / c)``; ``scale``:
    default 1 / sqrt(head_dim).  A query without a key gives zeros.  Returns q's shape and type.
    No value of ``lengths`` is read on the host, so the call can be captured in a CUDA graph; a table
    that is wide enough for 2^31 tiles of 32 keys and 8 or 16 query rows is refused.

    On CUDA weights are rounded to fp16 (11 bits down to 2^-29 of a row's largest, none below 2^-39);
    a score loses what is 28 binades under its key's largest block of K or 38 under its row's largest
    q; beside values of 2^79 and more, outputs lose what is below 2^-110.  Sums and the softmax's
    statistics are fp32."""
    one = q.dim() == 3
    if one:
        q = q.unsqueeze(2)
    if backend.native_for(q):
        out = backend.ext().fp4_kv_attention(
            q, pages, table, lengths, window,
            sink if sink is None or sink.dtype == torch.float32 else sink.float(), float(softcap or 0.0),
            q.shape[-1] ** -0.5 if scale is None else scale, error_word(q.device))
    else:
        if q.dim() != 4 or table.dim() != 2 or table.shape[0] != q.shape[0] or lengths.shape != q.shape[:1]:
            raise ValueError("q must be (B, H, T, head_dim), table (B, P), lengths (B,)")
        if table.dtype != torch.int32 or lengths.dtype != torch.int32:
            raise ValueError("table and lengths must be int32")
        if q.shape[1] % pages.shape[1] or window < 0 or (softcap or 0.0) < 0:
            raise ValueError("H must be a multiple of the K / V heads; window and softcap must not be negative")
        _check_table(pages, table, lengths, fp4_kv_page_rows(pages, q.shape[3]), q.shape[2], window)
        out = fp4_kv_attention_reference(q, pages, table, lengths, window=window, sink=sink, softcap=softcap,
                                         scale=scale)
    return out.squeeze(2) if one else out


__all__ = ["fp4_kv_attention", "fp4_kv_attention_reference", "fp4_kv_page_rows", "fp4_kv_read", "fp4_kv_slab_bytes",
           "fp4_kv_write"]
