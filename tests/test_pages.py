"""Pages of a cache without a GPU: the definition itself, and what the entry points refuse before any HIP call."""
import ctypes
import random

import numpy as np
import pytest
import torch

from pages_reference import Pages, entries
from ringattention_amd import paged
from ringattention_amd._lib import RingattnPagedPool, RingattnPages

OK, E_NULL, E_NPES, E_DIM, E_DTYPE, E_SEQLEN, E_SHAPE, E_WS, E_RANK, E_PLAN, E_HIP, E_ALLOC, E_ALIGN = range(13)


def test_the_definition_keeps_its_counts():
    """After any steps: counts are the entries that name a page, no row writes on a page that another one names."""
    rng = random.Random(1)
    for _ in range(60):
        rows, page = rng.randrange(1, 9), 16
        p = Pages(rng.randrange(1, 60), rows, rng.randrange(1, 10), page)
        for _ in range(12):
            before, parents = list(p.lens), None if rng.random() < 0.3 else [rng.randrange(-1, rows + 1) for _ in range(rows)]
            add = [rng.randrange(-40, 60) for _ in range(rows)]
            short, copies = p.update(parents, add)
            count = [0] * p.pages
            for b in range(rows):
                n = entries(p.lens[b], page)
                assert all(x >= 0 for x in p.table[b][:n]) and all(x == -1 for x in p.table[b][n:])
                for x in p.table[b][:n]:
                    count[x] += 1
            assert count == p.refs
            for b in range(rows):
                had = 0 if parents is not None and not 0 <= parents[b] < rows else before[b if parents is None else parents[b]]
                for j in range(had, p.lens[b]):   # tokens that are written next
                    assert p.refs[p.table[b][j // page]] == 1
                assert p.lens[b] == (had if short[b] else max(0, had + add[b]))
            assert len({t for _, t in copies}) == len(copies)
            if rng.random() < 0.3:
                n, moves, moved = p.compact()
                assert all(p.refs[:n]) and not any(p.refs[n:]) and sorted(x for x in moved if x >= 0) == list(range(n))


def test_refusals(ralib):
    memory = np.zeros(1 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    need = ralib.ringattn_pages_scratch_bytes(8, 3, 4)
    assert 0 < need <= 1 << 19
    for bad in ((0, 3, 4), (8, 0, 4), (8, 4097, 4), (8, 3, 0), (8, 4096, 2 ** 20), (8, -1, 4), (-8, 3, 4)):
        assert ralib.ringattn_pages_scratch_bytes(*bad) == 0, bad
    table = dict(refs=x, page_table=x, lens=x, table_stride=4, pages=8, rows=3, table_pages=4, page_size=16, scratch=x, scratch_bytes=need)
    pool = dict(k=x, v=x, scores=None, page_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, kv_heads=2, dim=64)

    def update(t=None, p=None, parents=None, add=None, missing=None, copies=None, none=False):
        t, p = RingattnPages(**dict(table, **(t or {}))), RingattnPagedPool(**dict(pool, **(p or {})))
        return ralib.ringattn_pages_update(ctypes.byref(t), None if none else ctypes.byref(p), parents, add, missing, copies, None)

    def compact(t=None, p=None, used=x, moved=None, moves=None, none=False):
        t, p = RingattnPages(**dict(table, **(t or {}))), RingattnPagedPool(**dict(pool, **(p or {})))
        return ralib.ringattn_pages_compact(ctypes.byref(t), None if none else ctypes.byref(p), used, moved, moves, None)

    for call in (update, compact):
        for bad, code in ((dict(refs=None), E_NULL), (dict(page_table=None), E_NULL), (dict(lens=None), E_NULL), (dict(refs=x + 4), E_ALIGN), (dict(lens=x + 2), E_ALIGN),
                          (dict(page_table=x + 1), E_ALIGN), (dict(pages=0), E_SHAPE), (dict(rows=0), E_SHAPE), (dict(rows=4097), E_SHAPE), (dict(table_pages=0), E_SHAPE),
                          (dict(page_size=24), E_SHAPE), (dict(page_size=8), E_SHAPE), (dict(page_size=2048), E_SHAPE), (dict(table_stride=3), E_SHAPE),
                          (dict(table_pages=2 ** 27, table_stride=2 ** 27), E_SHAPE), (dict(scratch=None), E_WS), (dict(scratch_bytes=need - 1), E_WS), (dict(scratch=x + 8), E_ALIGN)):
            assert call(t=bad) == code, bad
        for bad, code in ((dict(k=None), E_NULL), (dict(v=None), E_NULL), (dict(dim=96), E_DIM), (dict(kv_heads=0), E_SHAPE), (dict(token_stride=32), E_SHAPE),
                          (dict(page_stride=-8), E_SHAPE), (dict(head_stride=0), E_SHAPE), (dict(token_stride=68), E_ALIGN), (dict(k=x + 8), E_ALIGN), (dict(scores=x + 2), E_ALIGN),
                          (dict(page_stride=2 ** 39, kv_heads=65536), E_SHAPE)):
            assert call(p=bad) == code, bad
    assert update(parents=x + 1) == E_ALIGN and update(add=x + 2) == E_ALIGN and update(missing=x + 3) == E_ALIGN
    assert update(none=True) == E_NULL and compact(none=True) == E_NULL and update(copies=x + 4) == E_ALIGN and compact(moves=x + 4) == E_ALIGN
    assert compact(used=None) == E_NULL and compact(used=x + 2) == E_ALIGN and compact(moved=x + 2) == E_ALIGN

    def copy(f=None, t=None, from_pages=8, to_pages=8, page=16, pairs=x, n=0):
        f, t = RingattnPagedPool(**dict(pool, **(f or {}))), RingattnPagedPool(**dict(pool, **(t or {})))
        return ralib.ringattn_pages_copy(ctypes.byref(f), from_pages, ctypes.byref(t), to_pages, page, pairs, n, None)

    assert copy() == OK
    for bad, code in ((dict(f=dict(k=None)), E_NULL), (dict(t=dict(dim=128, token_stride=128)), E_SHAPE), (dict(t=dict(kv_heads=1)), E_SHAPE), (dict(t=dict(scores=x)), E_SHAPE),
                      (dict(from_pages=0), E_SHAPE), (dict(to_pages=-1), E_SHAPE), (dict(page=20), E_SHAPE), (dict(n=-1), E_SHAPE), (dict(pairs=None), E_NULL), (dict(pairs=x + 2), E_ALIGN)):
        assert copy(**bad) == code, bad


def test_python_refusals(ralib):
    for bad in (dict(pages=0), dict(rows=0), dict(rows=4097), dict(table_pages=0), dict(page_size=20), dict(page_size=0), dict(pages=2 ** 31), dict(table_pages=2 ** 27)):
        with pytest.raises(ValueError):
            paged.PagePool(**dict(dict(pages=4, rows=2, table_pages=3, page_size=16, device="cpu"), **bad))
    pool = paged.PagePool(4, 2, 3, 16, device="cpu")
    assert pool.page_table.shape == (2, 3) and (pool.page_table == -1).all() and not pool.refs.any() and not pool.lens.any()
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    for call in (lambda: pool.update(k, k), lambda: pool.compact(k, k), lambda: pool.update(k.float(), k.float()), lambda: pool.update(k[:, :, :8], k[:, :, :8]),
                 lambda: paged.copy_pages(k, k, k, k, torch.zeros(1, 2, dtype=torch.int32)), lambda: paged.copy_pages(k[0], k, k, k, torch.zeros(1, 2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()
