"""Page operators of a paged cache: reserve, fork, free and compact, on the device.

The state of a pool is ``table`` (S, P) int32 (row s: the page ids of sequence s in order, -1
behind the last), ``lengths`` (S,) int32 rows per sequence and ``refcount`` (n_pages,) int32: how
many table rows hold a page, 0 meaning free.  ``pool`` is any contiguous tensor (n_pages, ...):
bf16 rows, 4-bit pages of many layers; its bytes are only moved.  ``fork_pages`` and
``compact_pages`` return new state tensors and change ``pool`` in place, ``reserve_rows`` changes
the state in place (a captured decode step calls it); nothing is read on the host.

CPU tensors (and ``backend.eager_mode()``) take the definitions below; CUDA tensors run
``csrc/pages.cu``, where an index out of range or a pool with too few free pages is recorded and
raised by ``ops.gemm.check_errors``.
"""

from __future__ import annotations

import torch
from torch import Tensor

from saint_llm_b200.ops import backend
from saint_llm_b200.ops.gemm import error_word


def _check(pool: Tensor, table: Tensor, refcount: Tensor) -> None:
    if pool.dim() < 2 or not pool.is_contiguous():
        raise ValueError("pool must be a contiguous tensor (n_pages, ...)")
    if table.dim() != 2 or table.dtype != torch.int32 or refcount.dtype != torch.int32 or \
            refcount.shape != pool.shape[:1]:
        raise ValueError("table must be (rows, pages) int32 and refcount one int32 per page")
    if table.device != pool.device or refcount.device != pool.device:
        raise ValueError(f"pool, table and refcount must be on one device, got {pool.device} and {table.device}")


def reserve_rows(table: Tensor, lengths: Tensor, refcount: Tensor, rows: Tensor, count: int, *,
                 page_rows: int) -> Tensor:
    """Room for ``count`` more rows of each of the sequences ``rows`` (n,) int32, in place: pages are
    taken (the lowest free ones, in the order of ``rows``) where a row opens one, the lengths grow.
    Returns the rows' slots (n, count) int64 = page * page_rows + row.  ``rows`` must differ from one
    another.  With too few free pages, or a table too narrow, nothing changes, every slot is -1 (which
    writes skip) and an error is raised (on CUDA: by ``check_errors``)."""
    if backend.native_for(table):
        return backend.ext().reserve_rows(table, lengths, refcount, rows, count, page_rows, error_word(table.device))
    from saint_llm_b200.infer.paged_kv import PoolExhausted

    if table.dim() != 2 or rows.dim() != 1 or lengths.shape != table.shape[:1] or count <= 0 or page_rows <= 0:
        raise ValueError("table must be (rows, pages), lengths one per table row; count and page_rows positive")
    free = (refcount == 0).nonzero().flatten().tolist()
    taken = 0
    new: list[tuple[int, int, int]] = []
    for r in rows.tolist():
        if not 0 <= r < table.shape[0]:
            raise IndexError(f"row {r} of {table.shape[0]}")
        n = int(lengths[r])
        if n + count > table.shape[1] * page_rows:
            raise IndexError(f"{n + count} rows in a table for {table.shape[1] * page_rows}")
        for c in range(-(-n // page_rows), -(-(n + count) // page_rows)):
            if taken == len(free):
                raise PoolExhausted(f"{len(free)} of {len(refcount)} pages free, more needed")
            new.append((r, c, free[taken]))
            taken += 1
    for r, c, p in new:
        table[r, c] = p
        refcount[p] = 1
    pos = lengths[rows.long()].long().unsqueeze(1) + torch.arange(count, device=table.device)
    slots = table[rows.long()].long().gather(1, pos // page_rows) * page_rows + pos % page_rows
    lengths[rows.long()] += count
    return slots


def fork_pages(pool: Tensor, table: Tensor, lengths: Tensor, refcount: Tensor, parents: Tensor, children: Tensor, *,
               page_rows: int) -> tuple[Tensor, Tensor, Tensor]:
    """Table row ``children[i]`` becomes a copy of row ``parents[i]`` of the state as it was, for
    all i at once; a parent of -1 empties the row (its pages are freed when nobody else holds
    them).  Full pages are shared; a partly filled last page is copied into a free page, the
    lowest free ones in the order of i, so that parent and child can both append.  A child that is
    its own parent keeps its row.  ``children`` must differ from one another.

    One call serves best-of-n sampling (children: empty rows), a beam-search step (children:
    every row) and the end of requests (parents: -1).  Pages that this call frees are available to
    the next one.  With too few free pages nothing changes, and an error is raised (on CUDA: by
    ``check_errors``).  Returns (table, lengths, refcount)."""
    if backend.native_for(pool):
        return backend.ext().fork_pages(pool, table, lengths, refcount, parents, children, page_rows,
                                        error_word(pool.device))
    from saint_llm_b200.infer.paged_kv import PoolExhausted

    _check(pool, table, refcount)
    if parents.shape != children.shape or parents.dim() != 1 or lengths.shape != table.shape[:1] or page_rows <= 0:
        raise ValueError("parents and children must be vectors of one length, lengths one per table row")
    old, old_len = table.tolist(), lengths.tolist()
    new, new_len, refs = [list(r) for r in old], list(old_len), refcount.tolist()
    free = [p for p, n in enumerate(refs) if n == 0]
    copies = []
    for parent, child in zip(parents.tolist(), children.tolist(), strict=True):
        if not -1 <= parent < len(old) or not 0 <= child < len(old):
            raise IndexError(f"fork of row {parent} into row {child} of {len(old)}")
        if parent == child:
            continue
        row = list(old[parent]) if parent >= 0 else [-1] * table.shape[1]
        new_len[child] = old_len[parent] if parent >= 0 else 0
        if new_len[child] % page_rows:
            if len(copies) == len(free):
                raise PoolExhausted(f"{len(free)} of {len(refs)} pages free, more needed")
            tail = new_len[child] // page_rows
            copies.append((row[tail], free[len(copies)]))
            row[tail] = copies[-1][1]
        for p in old[child]:
            if p >= 0:
                refs[p] -= 1
        for p in row:
            if p >= 0:
                refs[p] += 1
        new[child] = row
    for src, dst in copies:
        pool[dst] = pool[src]
    dev = table.device
    return (torch.tensor(new, dtype=torch.int32, device=dev).view(table.shape),
            torch.tensor(new_len, dtype=torch.int32, device=dev), torch.tensor(refs, dtype=torch.int32, device=dev))


def compact_pages(pool: Tensor, table: Tensor, refcount: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """Move the pages in use to the front of the pool.  With n pages in use, those with an id of n
    or more move into the free ids below n, both in ascending order; the table's ids follow (an id
    of a page that is not in use becomes -1).  Returns (table, refcount, n): afterwards the pages
    n and up are free.  Contents of pages that are free afterwards are unspecified."""
    if backend.native_for(pool):
        return backend.ext().compact_pages(pool, table, refcount, error_word(pool.device))
    _check(pool, table, refcount)
    used = refcount > 0
    n = used.sum()
    page = torch.arange(len(refcount), device=refcount.device)
    hole, late = ((~used) & (page < n)).nonzero().flatten(), (used & (page >= n)).nonzero().flatten()
    where = torch.where(used, page, -1)
    where[late] = hole
    pool[hole] = pool[late]
    refs = torch.where(page < n, refcount, 0)
    refs[hole] = refcount[late]
    ids = table.long()
    if bool((ids >= len(refcount)).any()):
        raise IndexError("the table names a page outside the pool")
    return torch.where(ids >= 0, where[ids.clamp(min=0)].int(), -1).int(), refs, n.int()


__all__ = ["compact_pages", "fork_pages", "reserve_rows"]
