"""The paged cache's parameters without a GPU: what is taken and what is refused before any HIP call."""
import ctypes

import pytest

from ringattention_amd import paged
from ringattention_amd._lib import RingattnPagedCache
from test_paged import E_SHAPE, OK, memory, params  # noqa: F401  (memory: a fixture)


def test_flags(ralib, memory):  # noqa: F811
    base, size = memory
    for flags, code in ((paged.FLAG_PAGED_PARTIALS, OK), (paged.FLAG_PAGED_KEEP_PRESENT, OK), (5, OK), (2, E_SHAPE), (6, E_SHAPE), (8, E_SHAPE), (-1, E_SHAPE)):
        h = ctypes.c_void_p()
        assert ralib.ringattn_paged_plan_create(ctypes.byref(params(flags=flags)), ctypes.c_void_p(base), size, ctypes.byref(h)) == code, flags
        if code == OK:
            assert ralib.ringattn_paged_plan_destroy(h) == OK
    plan = paged.PagedAttention(8, 64, kv_heads=2, page_size=16, workspace=memory, keep_present=True)
    assert plan.params.flags == 4
    plan.close()


def test_numbers_beyond_32_bits(memory):  # noqa: F811
    """They are refused, not taken for what is left of them: a window of 2^32 + 5 is none of 5."""
    for bad in (dict(window=2 ** 32 + 5), dict(window=5, sinks=2 ** 32), dict(window=-2 ** 32 + 5), dict(max_tokens=2 ** 32 + 64), dict(max_batch=2 ** 32 + 4),
                dict(page_size=2 ** 32 + 16), dict(kv_heads=2 ** 32 + 2)):
        with pytest.raises(ValueError, match="32 bits"):
            paged.PagedAttention(8, 64, **dict(dict(kv_heads=2, page_size=16, workspace=memory), **bad))
    with pytest.raises(ValueError, match="32 bits"):
        paged.PagedAttention(8, 2 ** 32 + 64, kv_heads=2, page_size=16, workspace=memory)


def test_pools_beyond_64_bits(ralib, memory):  # noqa: F811
    """A pool whose last page would lie past 2^60 elements is none, whatever each of its strides is."""
    base, size = memory
    h = ctypes.c_void_p()
    assert ralib.ringattn_paged_plan_create(ctypes.byref(params()), ctypes.c_void_p(base), size, ctypes.byref(h)) == OK
    for pages, page_stride, code in ((2 ** 31 - 1, 2 ** 38, E_SHAPE), (2 ** 22, 2 ** 39, E_SHAPE), (2 ** 21, 2 ** 39, OK), (2 ** 31 - 1, 2 ** 29, OK)):
        c = ctypes.byref(RingattnPagedCache(k=base, v=base, page_stride=page_stride, head_stride=1024, token_stride=64, pages=pages, table_pages=4,
                                            table_stride=4, page_table=base, kv_lens=base, q_starts=base, batch=0))
        assert ralib.ringattn_paged_fwd(h, c, base, 5, 512, 64, base, 512, 64, base, None) == code, (pages, page_stride)
        assert ralib.ringattn_paged_evict(h, c, base, base, 2, 2, 20, 2, 3, base, base, None) == code
    assert ralib.ringattn_paged_plan_destroy(h) == OK
