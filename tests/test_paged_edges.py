"""The paged cache's parameters without a GPU: what is taken and what is refused before any HIP call."""
import ctypes

import pytest

from ringattention_amd import paged
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
