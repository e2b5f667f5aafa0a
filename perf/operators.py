"""The paged 4-bit KV cache and its page operators: plain forms, inputs and sizes.

Operators (``case["op"]``):

* ``attend``: attention of T query tokens per sequence over K / V held in 4 bits in pages;
* ``store``: K / V rows quantised into pages, and the same rows read back;
* ``fork``: rows of a block table replaced by other rows (shared pages, copied tails, freed pages);
* ``compact``: live pages moved to the front of the pool, tables renumbered.

Page format: ``pages`` (n_pages, kv_heads, slab) uint8; a slab is the K codes (page_rows x
head_dim / 2 bytes), the V codes, the K scales (page_rows x head_dim / 32 bytes) and the V
scales.  Byte j of a row's codes holds dim 2j in its low and dim 2j + 1 in its high four bits
(E2M1: sign, two exponent bits, one mantissa bit); every 32 dims share a scale 2^(byte - 127),
byte 255 being NaN.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LIMITS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # midpoints: a tie goes to the smaller magnitude


# --------------------------------------------------------------------------- cases
def _attend(name, b, h, hk, d, t, n, r, window, sink, softcap, dtype):
    return {"name": name, "op": "attend", "batch": b, "heads": h, "kv_heads": hk, "head_dim": d, "tokens": t,
            "max_len": n, "page_rows": r, "window": window, "sink": sink, "softcap": softcap, "dtype": dtype}


def _store(name, n, hk, d, r, dtype):
    return {"name": name, "op": "store", "rows": n, "kv_heads": hk, "head_dim": d, "page_rows": r, "dtype": dtype}


def _fork(name, seqs, max_pages, forks, r, n_pages, kind, page_bytes):
    return {"name": name, "op": "fork", "seqs": seqs, "max_pages": max_pages, "forks": forks, "page_rows": r,
            "n_pages": n_pages, "kind": kind, "page_bytes": page_bytes}


def _compact(name, seqs, max_pages, n_pages, live, kind, page_bytes):
    return {"name": name, "op": "compact", "seqs": seqs, "max_pages": max_pages, "n_pages": n_pages, "live": live,
            "kind": kind, "page_bytes": page_bytes}


def listed():
    return [
        # one chat request in its first thousand tokens, 16 heads of 128 over one K/V head: latency
        _attend("attend_one", 1, 16, 1, 128, 1, 777, 64, 0, True, 0.0, "bf16"),
        # the decode benchmark's batch: 64 requests of 4096 + 512 tokens, window 4096
        _attend("attend_batch64", 64, 16, 1, 128, 1, 4608, 64, 4096, True, 0.0, "bf16"),
        # four long documents with grouped heads: the cache itself is the traffic
        _attend("attend_long", 4, 32, 8, 128, 1, 131072, 64, 0, False, 0.0, "bf16"),
        # five drafted tokens verified per request, 12 heads of 64 (small_flash), half precision, softcap
        _attend("attend_verify", 24, 12, 1, 64, 5, 2001, 16, 0, True, 30.0, "f16"),
        # a prefill chunk of 256 tokens over what is cached already
        _attend("attend_chunk", 4, 16, 1, 128, 256, 8192, 128, 0, True, 0.0, "bf16"),
        # one decode step of 64 requests stores one row each
        _store("store_step", 64, 1, 128, 64, "bf16"),
        # a prefill step: 64 requests, chunks of 256 tokens and a few odd ones
        _store("store_chunk", 16411, 1, 128, 64, "bf16"),
        # a long grouped-head prompt kept in 32 bits, small pages
        _store("store_grouped", 65537, 8, 128, 16, "f32"),
        # one beam-search step: 32 beams of one layer's bf16 pool
        _fork("fork_beams", 32, 64, 32, 64, 2048, "bf16", 16384),
        # sixteen samples each of four prompts, a page holding 28 layers in 4 bits
        _fork("fork_samples", 128, 128, 64, 64, 2048, "fp4", 28 * 8704),
        # a small bf16 pool after some requests finished
        _compact("compact_small", 16, 64, 512, 0.5, "bf16", 16384),
        # a gigabyte of 28-layer pages, two fifths of them live
        _compact("compact_serving", 256, 64, 4096, 0.4, "fp4", 28 * 8704),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["attend", "attend", "store", "fork", "compact"])
    if op == "attend":
        t = rng.choice([1, 1, 1, 1, rng.randint(2, 8), rng.randint(2, 8), _log(rng, 9, 256)])
        hk = rng.choice([1, 1, 2, 4, 8])
        g = rng.choice([12, 16, 16, 32, 64]) if hk == 1 else rng.choice([1, 2, 3, 4, 7, 8])
        d = rng.choice([64, 128, 128])
        b = _log(rng, 1, 64)
        top = min(4 * 8 * 131072 * 128 // (b * hk * d), 4 * 16 * 256 * 8192 * 128 // (b * hk * g * t * d), 131072)
        n = _log(rng, max(1, min(t, top)), max(t, top))
        c = _attend("", b, g * hk, hk, d, t, n, rng.choice([16, 32, 64, 128]),
                    rng.choice([0, 0, max(1, n // 2), 128]), rng.random() < 0.5, rng.choice([0.0, 0.0, 50.0]),
                    rng.choice(["bf16", "bf16", "f16"]))
    elif op == "store":
        hk, d = rng.choice([1, 1, 2, 8]), rng.choice([64, 128])
        c = _store("", _log(rng, 1, 65537 * 8 // hk // 2), hk, d, rng.choice([16, 32, 64, 128]),
                   rng.choice(["bf16", "bf16", "f16", "f32"]))
    else:
        r, d, hk, layers = rng.choice([16, 32, 64, 128]), rng.choice([64, 128]), rng.choice([1, 1, 2]), _log(rng, 1, 28)
        kind = rng.choice(["bf16", "fp4"])
        size = r * d * 2 if kind == "bf16" else layers * hk * (r * d * 17 // 16)
        n_pages = _log(rng, 64, max(65, min(8192, 900_000_000 // size)))
        seqs = max(1, min(256, _log(rng, 2, max(3, n_pages // 4))))
        max_pages = max(1, min(128, n_pages // (2 * seqs)))
        if op == "fork":
            c = _fork("", seqs, max_pages, rng.randint(1, min(64, seqs)), r, n_pages, kind, size)
        else:
            c = _compact("", seqs, max_pages, n_pages, round(rng.uniform(0.1, 0.9), 3), kind, size)
    del c["name"]
    return c


# --------------------------------------------------------------------------- the format, plainly
def _slab(r, d):
    return r * d + r * d // 16


def _scale_of(byte):
    """2^(byte - 127) in 32 bits, 255 being NaN."""
    s = (byte.int() << 23).view(torch.float32)
    return torch.where(byte == 255, torch.full_like(s, float("nan")), s)


def _quantise(x):
    """x (..., d) -> codes (..., d) uint8 below 16 and scale bytes (..., d / 32)."""
    blocks = x.float().unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1): the smallest exponent with amax <= 6 * 2^exponent
    exp = torch.where(amax > 0, e - 3 + (m > 0.75).int(), torch.full_like(e, -126)).clamp(-126, 126)
    byte = torch.where(torch.isfinite(amax), exp + 127, torch.full_like(exp, 255))
    mag = blocks.abs() * ((127 - exp) << 23).view(torch.float32).unsqueeze(-1)
    code = torch.zeros_like(mag, dtype=torch.uint8)
    for limit in LIMITS:
        code += mag > limit
    code = torch.where((blocks < 0) & (code > 0), code + 8, code)
    return code.flatten(-2), byte.to(torch.uint8)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _unpack(packed):
    """packed (..., d / 2) uint8 -> values (..., d) in 32 bits."""
    code = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=packed.device)
    return levels[code.int()]


def _parts(pages, r, d):
    """Views of a pages tensor (n, heads, slab): K codes, V codes (n, heads, r, d/2), K, V scales (n, heads, r, d/32)."""
    c, s = r * d // 2, r * d // 32
    cut = [pages[..., 0:c], pages[..., c:2 * c], pages[..., 2 * c:2 * c + s], pages[..., 2 * c + s:2 * c + 2 * s]]
    return [p.unflatten(-1, (r, -1)) for p in cut]


def _put(pages, r, d, slots, k, v):
    """Rows k, v (N, heads, d) written at ``slots`` (N,) = page * r + row."""
    kc, vc, ks, vs = _parts(pages, r, d)
    page, row = slots // r, slots % r
    code, byte = _quantise(k)
    kc[page, :, row], ks[page, :, row] = _pack(code), byte
    code, byte = _quantise(v)
    vc[page, :, row], vs[page, :, row] = _pack(code), byte


def _values(codes, scales):
    return (_unpack(codes).unflatten(-1, (-1, BLOCK)) * _scale_of(scales).unsqueeze(-1)).flatten(-2)


# --------------------------------------------------------------------------- inputs
def _rows(n, hk, d, gen):
    """K rows with a few strong channels, V rows of differing size: what caches hold."""
    k = torch.randn(n, hk, d, generator=gen, device=DEV)
    k[..., ::37] *= 6.0
    v = torch.randn(n, hk, d, generator=gen, device=DEV)
    v *= torch.exp(0.7 * torch.randn(n, hk, 1, generator=gen, device=DEV))
    return k, v


def _lengths(case, rng):
    """Ragged lengths: one the longest, and in a batch of four or more one empty and one of one token."""
    b, n = case["batch"], case["max_len"]
    lens = [n] + [rng.randint(max(1, n // 2), n) for _ in range(b - 1)]
    if b >= 4:
        lens[1], lens[2] = 0, 1
    return lens


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    op = case["op"]
    if op == "attend":
        b, hk, d, r = case["batch"], case["kv_heads"], case["head_dim"], case["page_rows"]
        dtype = DTYPES[case["dtype"]]
        lens = _lengths(case, rng)
        counts = [-(-n // r) for n in lens]
        width = max(counts)
        n_pages = sum(counts) + 3
        # pages in no order; what no row was written to holds anything at all
        order = torch.randperm(n_pages, generator=gen, device=DEV).int()
        pages = torch.randint(0, 256, (n_pages, hk, _slab(r, d)), generator=gen, device=DEV, dtype=torch.uint8)
        table = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(lens):
            table[i, :counts[i]] = order[at:at + counts[i]]
            at += counts[i]
            for lo in range(0, n, 32768):
                pos = torch.arange(lo, min(n, lo + 32768), device=DEV)
                k, v = _rows(len(pos), hk, d, gen)
                _put(pages, r, d, table[i, pos // r].long() * r + pos % r, k, v)
        q = (1.5 * torch.randn(b, case["heads"], case["tokens"], d, generator=gen, device=DEV)).to(dtype)
        sink = torch.randn(case["heads"], generator=gen, device=DEV) if case["sink"] else None
        return {"case": case, "q": q, "pages": pages, "table": table, "sink": sink,
                "lengths": torch.tensor(lens, dtype=torch.int32, device=DEV)}
    if op == "store":
        n, hk, d, r = case["rows"], case["kv_heads"], case["head_dim"], case["page_rows"]
        n_pages = -(-n // r) + 8
        pages = torch.randint(0, 256, (n_pages, hk, _slab(r, d)), generator=gen, device=DEV, dtype=torch.uint8)
        # rows follow one another within a page, pages in no order
        page = torch.randperm(n_pages, generator=gen, device=DEV)
        pos = torch.arange(n, device=DEV)
        k, v = _rows(n, hk, d, gen)
        dtype = DTYPES[case["dtype"]]
        return {"case": case, "k": k.to(dtype), "v": v.to(dtype), "pages": pages, "slots": page[pos // r] * r + pos % r}
    s, p, n_pages = case["seqs"], case["max_pages"], case["n_pages"]
    if case["kind"] == "bf16":
        pool = torch.randn(n_pages, case["page_bytes"] // 2, generator=gen, device=DEV, dtype=torch.bfloat16)
    else:
        pool = torch.randint(0, 256, (n_pages, case["page_bytes"]), generator=gen, device=DEV, dtype=torch.uint8)
    order = torch.randperm(n_pages, generator=gen, device=DEV).tolist()
    table = [[-1] * p for _ in range(s)]
    refs = [0] * n_pages
    if op == "fork":
        r, f = case["page_rows"], case["forks"]
        lens = [rng.randint(1, p * r) for _ in range(s)]
        spare = n_pages - f
        for i in range(s):  # what does not fit beside the copies to come gets a shorter row
            need = -(-lens[i] // r)
            if need > spare:
                need, lens[i] = max(0, spare), max(0, spare) * r
            spare -= need
            table[i][:need] = [order.pop() for _ in range(need)]
            for page in table[i][:need]:
                refs[page] += 1
        children = rng.sample(range(s), f)
        few = rng.sample(range(s), min(s, max(1, f // 16)))
        parents = [rng.choice(few) if f < s else rng.randrange(s) for _ in range(f)]
        if f > 8:
            parents[3] = -1  # a finished request is freed in the same step
        ints = {"lengths": lens, "parents": parents, "children": children}
    else:
        want = max(1, int(case["live"] * n_pages))
        for i in range(s):
            need = min(want, rng.randint(1, p))
            want -= need
            table[i][:need] = [order.pop() for _ in range(need)]
            if i % 5 == 4:  # a fork of the row before it: shared pages
                shared = [x for x in table[i - 1][:need // 2] if x >= 0]
                table[i][:len(shared)] = shared
            for page in table[i]:
                if page >= 0:
                    refs[page] += 1
        ints = {}
    state = {"case": case, "pool": pool, "table": torch.tensor(table, dtype=torch.int32, device=DEV),
             "refcount": torch.tensor(refs, dtype=torch.int32, device=DEV)}
    state.update({k: torch.tensor(v, dtype=torch.int32, device=DEV) for k, v in ints.items()})
    return state


# --------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return _own(op, case, state)
    return {"attend": _plain_attend, "store": _plain_store, "fork": _plain_fork, "compact": _plain_compact}[op](state)


def _own(op, case, s):
    from saint_llm_b200.ops import fp4_kv, pages

    if op == "attend":
        return fp4_kv.fp4_kv_attention(s["q"], s["pages"], s["table"], s["lengths"], window=case["window"],
                                       sink=s["sink"], softcap=case["softcap"] or None)
    if op == "store":
        fp4_kv.fp4_kv_write(s["k"], s["v"], s["pages"], s["slots"])
        return fp4_kv.fp4_kv_read(s["pages"], s["slots"], head_dim=case["head_dim"], dtype=s["k"].dtype)
    if op == "fork":
        return s["pool"], *pages.fork_pages(s["pool"], s["table"], s["lengths"], s["refcount"], s["parents"],
                                            s["children"], page_rows=case["page_rows"])
    return s["pool"], *pages.compact_pages(s["pool"], s["table"], s["refcount"])


def _plain_attend(s):
    case, q, table = s["case"], s["q"].float(), s["table"]
    r, d, hk, t = case["page_rows"], case["head_dim"], case["kv_heads"], case["tokens"]
    b, h, g = case["batch"], case["heads"], case["heads"] // case["kv_heads"]
    kc, vc, ks, vs = _parts(s["pages"][table.clamp(min=0)], r, d)  # (B, P, Hk, r, ...)
    n = table.shape[1] * r
    k = _values(kc, ks).transpose(1, 2).reshape(b, hk, n, d)
    v = _values(vc, vs).transpose(1, 2).reshape(b, hk, n, d)
    lens = s["lengths"].view(b, 1, 1)
    key = torch.arange(n, device=q.device)
    pos = lens - t + torch.arange(t, device=q.device).view(1, t, 1)
    seen = (key <= pos) & (key < lens)  # (B, T, n)
    if case["window"]:
        seen = seen & (key > pos - case["window"])
    seen = seen.view(b, 1, 1, t, n)
    # nothing that a row may not see reaches a product: unwritten rows may hold NaN
    live = (key < lens).view(b, 1, n, 1)
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    x = (q.view(b, hk, g * t, d) @ k.transpose(-1, -2)).view(b, hk, g, t, n) / math.sqrt(d)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    x = torch.where(seen, x, float("-inf"))
    m = x.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, hk, g, 1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - m)
    o = (p.view(b, hk, g * t, n) @ v).view(b, hk, g, t, d) / torch.where(total > 0, total, 1.0)
    return o.view(b, h, t, d).to(s["q"].dtype)


def _plain_store(s):
    case, slots = s["case"], s["slots"]
    r, d = case["page_rows"], case["head_dim"]
    _put(s["pages"], r, d, slots, s["k"], s["v"])
    kc, vc, ks, vs = (part[slots // r, :, slots % r] for part in _parts(s["pages"], r, d))
    return _values(kc, ks).to(s["k"].dtype), _values(vc, vs).to(s["k"].dtype)


def _plain_fork(s):
    case, pool, table, lengths, refs = s["case"], s["pool"], s["table"], s["lengths"], s["refcount"]
    r, p = case["page_rows"], case["max_pages"]
    child, parent = s["children"].long(), s["parents"].long()
    takes = parent >= 0
    src = parent.clamp(min=0)
    moved = parent != child
    length = torch.where(takes, lengths[src], 0)
    rows = torch.where(takes.unsqueeze(1), table[src], -1)
    copied = takes & moved & (length % r != 0)
    tail = (length // r).long()
    free = (refs == 0).nonzero().flatten()
    fresh = free[torch.where(copied, copied.long().cumsum(0) - 1, 0).clamp(max=len(free) - 1)].int()
    col = torch.arange(p, device=table.device)
    is_tail = copied.unsqueeze(1) & (col == tail.unsqueeze(1))
    old_tail = table[src, tail.clamp(max=p - 1)].long()
    new_table, new_lengths, new_refs = table.clone(), lengths.clone(), refs.clone()
    new_table[child] = torch.where(is_tail, fresh.unsqueeze(1), rows)
    new_lengths[child] = length
    gone = table[child][moved.unsqueeze(1) & (table[child] >= 0)].long()
    kept = rows[moved.unsqueeze(1) & (rows >= 0) & ~is_tail].long()
    new_refs.index_add_(0, gone, torch.full_like(gone, -1).int())
    new_refs.index_add_(0, kept, torch.ones_like(kept).int())
    new_refs[fresh[copied].long()] = 1
    pool[fresh[copied].long()] = pool[old_tail[copied]]
    return pool, new_table, new_lengths, new_refs


def _plain_compact(s):
    pool, table, refs = s["pool"], s["table"], s["refcount"]
    live = refs > 0
    n_live = live.sum()
    page = torch.arange(len(refs), device=refs.device)
    hole = (~live & (page < n_live)).nonzero().flatten()
    late = (live & (page >= n_live)).nonzero().flatten()
    where = torch.where(live, page, -1)
    where[late] = hole
    pool[hole] = pool[late]
    new_refs = torch.where(page < n_live, refs, 0)
    new_refs[hole] = refs[late]
    new_table = torch.where(table >= 0, where[table.clamp(min=0).long()].int(), -1)
    return pool, new_table, new_refs, n_live.int()


# --------------------------------------------------------------------------- the definition in 64 bits
def _power(e):
    """2^e exactly, from the bits of a 64-bit number."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(codes, scales):
    """Sign, exponent and mantissa bits of each four bits, by arithmetic."""
    c = torch.stack((codes.long() % 16, codes.long() // 16), -1).reshape(*codes.shape[:-1], -1)
    two, half = c // 2 % 4, (c % 2).double() / 2
    mag = torch.where(two == 0, half, (1 + half) * _power(two - 1))
    mag = torch.where(c >= 8, -mag, mag)
    factor = _power(scales.long() - 127).masked_fill(scales == 255, float("nan"))
    return mag * factor.repeat_interleave(BLOCK, -1)


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers and copies
    s = prepare(case, seed)
    r, d, hk = case["page_rows"], case["head_dim"], case["kv_heads"]
    if case["op"] == "store":
        out = []
        for x in (s["k"], s["v"]):
            y = x.double().reshape(*x.shape[:-1], -1, BLOCK)
            amax = y.abs().amax(-1, keepdim=True)
            step = _power(torch.ceil(torch.log2((amax / 6.0).clamp(min=1e-300))).clamp(-126, 126))
            step = torch.where(amax / 6 > step, 2 * step, torch.where(amax / 6 <= step / 2, step / 2, step))
            levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
            # nearest level, the lower one of two that are equally near
            near = torch.searchsorted((levels[1:] + levels[:-1]) / 2, (y.abs() / step).contiguous())
            out.append((torch.sign(y) * levels[near] * step).reshape(x.shape))
        return tuple(out)
    g, t = case["heads"] // hk, case["tokens"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    slab = s["pages"].view(-1, hk, _slab(r, d))
    half, few = r * d // 2, r * d // 32
    for b, n in enumerate(s["lengths"].tolist()):
        ids = s["table"][b, :-(-n // r)].long() if n else None
        for j in range(hk):
            mine = slab[ids, j] if n else None
            k = v = None
            if n:
                k = _decode64(mine[:, :half].reshape(-1, d // 2), mine[:, 2 * half:2 * half + few].reshape(-1, d // 32))[:n]
                v = _decode64(mine[:, half:2 * half].reshape(-1, d // 2), mine[:, 2 * half + few:].reshape(-1, d // 32))[:n]
            for i in range(t):
                pos = n - t + i
                first = max(0, pos - case["window"] + 1) if case["window"] else 0
                if pos < first:
                    continue
                x = s["q"][b, j * g:(j + 1) * g, i].double() @ k[first:pos + 1].T / math.sqrt(d)
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                if s["sink"] is not None:
                    x = torch.cat([x, s["sink"][j * g:(j + 1) * g, None].double()], -1)
                w = torch.softmax(x, -1)[:, :pos + 1 - first]
                out[b, j * g:(j + 1) * g, i] = w @ v[first:pos + 1]
    return out


# --------------------------------------------------------------------------- what one pass cannot do without
def work(case):
    op = case["op"]
    if op == "store":
        values = case["rows"] * case["kv_heads"] * case["head_dim"] * 2
        size = DTYPES[case["dtype"]].itemsize
        held = values * 17 / 32
        return {"bytes": 2 * values * size + 2 * held + 8 * case["rows"], "flops": 0}
    if op == "attend":
        rng = random.Random(0)
        t, w, pairs, rows = case["tokens"], case["window"], 0, 0
        for n in _lengths(case, rng):
            seen = min(n, w + t - 1) if w else n
            rows += seen
            for i in range(t):
                at = n - t + i + 1
                pairs += max(0, min(at, w) if w else at)
        d = case["head_dim"]
        held = rows * case["kv_heads"] * d * 17 / 16
        q = case["batch"] * case["heads"] * t * d * 2
        return {"bytes": held + 2 * q, "flops": 4 * pairs * case["heads"] * d}
    if op == "fork":  # nearly every fork copies a tail page
        return {"bytes": 2 * case["forks"] * case["page_bytes"] + 8 * case["seqs"] * case["max_pages"]
                + 8 * case["n_pages"], "flops": 0}
    live = min(case["live"] * case["n_pages"], case["seqs"] * (case["max_pages"] + 1) / 2)
    moved = live * (1 - live / case["n_pages"])
    return {"bytes": 2 * moved * case["page_bytes"] + 8 * case["seqs"] * case["max_pages"] + 8 * case["n_pages"],
            "flops": 0}
