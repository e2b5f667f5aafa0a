"""Plain 64-bit implementations of the 4-bit K / V cache, one row and one code at a time, written
apart from the package's own definitions."""

import math

import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """x (..., d) float64 -> codes (..., d), scale bytes (..., d/32), values (..., d)."""
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(blocks).max(-1, keepdims=True)
    e = np.full(amax.shape, -126)
    for k in range(-126, 127):  # the smallest exponent with amax <= 6 * 2^e
        e = np.where(amax > 6.0 * 2.0 ** k, k + 1, e)
    e = np.minimum(e, 126)
    bad = ~np.isfinite(amax)
    with np.errstate(invalid="ignore"):
        ratio = np.where(bad, 0.0, np.abs(blocks) / 2.0 ** e)
        sign = blocks < 0
    distance = np.abs(ratio[..., None] - LEVELS)
    code = distance.argmin(-1)  # the first of two that are equally near is the smaller
    value = np.where(bad, np.nan, np.where(sign, -1.0, 1.0) * LEVELS[code] * 2.0 ** e)
    code = np.where(sign & (code > 0), code + 8, code)
    byte = np.where(bad, 255, e + 127)[..., 0]
    return code.reshape(x.shape), byte, value.reshape(x.shape)


def put(pages: np.ndarray, rows: int, slot: int, k: np.ndarray, v: np.ndarray) -> None:
    """Row k, v (heads, d) into ``pages`` (n, heads, slab) uint8 at ``slot``, byte by byte."""
    page, r = divmod(int(slot), rows)
    d = k.shape[1]
    for which, x in enumerate((k, v)):
        code, byte, _ = quantise(x)
        for h in range(x.shape[0]):
            slab = pages[page, h]
            at = which * rows * d // 2 + r * d // 2
            for j in range(d // 2):
                slab[at + j] = code[h, 2 * j] | (code[h, 2 * j + 1] << 4)
            at = rows * d + which * rows * d // 32 + r * d // 32
            slab[at:at + d // 32] = byte[h]


def rows_of(pages: torch.Tensor, rows: int, d: int, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """K, V (N, heads, d) float64 at ``slots``."""
    page, r = slots // rows, slots % rows
    out = []
    for which in range(2):
        code = pages[page, :, which * rows * d // 2:(which + 1) * rows * d // 2].unflatten(-1, (rows, -1))
        lo = rows * d + which * rows * d // 32
        byte = pages[page, :, lo:lo + rows * d // 32].unflatten(-1, (rows, -1))
        n = torch.arange(len(slots), device=slots.device)
        code, byte = code[n, :, r].long(), byte[n, :, r].long()
        c = torch.stack([code % 16, code // 16], -1).flatten(-2)
        mag = torch.tensor(LEVELS, device=c.device)[c % 8] * torch.where(c >= 8, -1.0, 1.0)
        scale = ((byte + (1023 - 127)) << 52).view(torch.float64)
        scale = torch.where(byte == 255, float("nan"), scale)
        out.append(mag * scale.repeat_interleave(32, -1))
    return out[0], out[1]


def attention(q, pages, table, lengths, rows, *, window=0, sink=None, softcap=None, scale=None):
    """(out, size, score, floor): the definition in 64 bits; sum p |v| / sum p, the size that
    rounding errors of the weights scale with; the largest scale * sum |q k|, that errors of the
    scores scale with; keys * largest |v|, that the loss of the smallest weights scales with.
    q (B, H, T, d)."""
    b_, h_, t_, d = q.shape
    hk = pages.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    score = torch.zeros(*q.shape[:3], 1, dtype=torch.float64, device=q.device)
    floor = torch.zeros_like(score)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    for b in range(b_):
        n = int(lengths[b])
        if n == 0:
            continue
        pos = torch.arange(n, device=q.device)
        slots = table[b, pos // rows].long() * rows + pos % rows
        k, v = rows_of(pages, rows, d, slots)
        for h in range(h_):
            kh, vh = k[:, h // (h_ // hk)], v[:, h // (h_ // hk)]
            for t in range(t_):
                at = n - t_ + t
                lo = max(0, at - window + 1) if window else 0
                if at < lo:
                    continue
                s = (kh[lo:at + 1] @ q[b, h, t].double()) * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                score[b, h, t] = (kh[lo:at + 1].abs() @ q[b, h, t].double().abs()).max() * abs(scale)
                floor[b, h, t] = len(s) * vh[lo:at + 1].abs().max()
                m = s.max()
                if sink is not None:
                    m = torch.maximum(m, sink[h].double())
                p = torch.exp(s - m)
                total = p.sum() + (torch.exp(sink[h].double() - m) if sink is not None else 0.0)
                out[b, h, t] = p @ vh[lo:at + 1] / total
                size[b, h, t] = p @ vh[lo:at + 1].abs() / total
    return out, size, score, floor


def bound(out, size, score, floor, dtype):
    """How far an output may be from ``out``: half a unit of its type (bf16 2^-8, fp16 2^-11 of
    the value; the smallest are spaced by 2^-133 and 2^-24); the weights' rounding to fp16
    (2^-11), in numerator and denominator, with a quarter more for 32-bit sums and exp; the
    scores' error, 2^-20 of their products' sizes (eight 32-bit partial sums), which a weight
    repeats, in numerator and denominator; and the smallest weights, spaced by 2^-39 of the
    largest (fp16 holds them times 2^15)."""
    unit, tiny = (2.0 ** -8, 2.0 ** -134) if dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -25)
    return unit * out.abs() + tiny + (2.5 * 2.0 ** -11 + 2.0 ** -19 * score) * size + 2.0 ** -40 * floor


def filled(lens, *, hk, d, rows, gen, device, spare=2, spread=None):
    """Pages with random rows for sequences of ``lens`` (written through the package), in shuffled
    pages whose other bytes are random.  Returns pages, table, lengths."""
    from saint_llm_b200.ops.fp4_kv import fp4_kv_slab_bytes, fp4_kv_write

    counts = [-(-n // rows) for n in lens]
    n_pages = sum(counts) + spare
    pages = torch.randint(0, 256, (n_pages, hk, fp4_kv_slab_bytes(rows, d)), generator=gen, dtype=torch.uint8)
    order = torch.randperm(n_pages, generator=gen).int()
    table = torch.full((len(lens), max(1, *counts)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    slots = [table[i, torch.arange(n) // rows].long() * rows + torch.arange(n) % rows for i, n in enumerate(lens)]
    slots = torch.cat(slots) if slots else torch.empty(0, dtype=torch.long)
    k = torch.randn(len(slots), hk, d, generator=gen)
    v = torch.randn(len(slots), hk, d, generator=gen)
    if spread is not None:
        v = v * 2.0 ** torch.randint(-spread, spread + 1, (len(slots), hk, 1), generator=gen)
    pages = pages.to(device)
    fp4_kv_write(k.to(device), v.to(device), pages, slots.to(device))
    return pages, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)
