"""Scored attention over the paged cache without a GPU: what the C entry points refuse before any HIP call."""
import ctypes

import numpy as np
import pytest
import torch

from ringattention_amd import paged
from ringattention_amd._lib import RingattnPagedCache, RingattnPagedScoring
from test_paged import params

OK, E_NULL, E_NPES, E_DIM, E_DTYPE, E_SEQLEN, E_SHAPE, E_WS, E_RANK, E_PLAN, E_HIP, E_ALLOC, E_ALIGN = range(13)


def test_scoring_refusals(ralib):
    memory = np.zeros(160 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    plans = {}
    for causal in (1, 0):
        h = ctypes.c_void_p()
        assert ralib.ringattn_paged_plan_create(ctypes.byref(params(causal=causal)), ctypes.c_void_p(x), (160 << 20) - 16, ctypes.byref(h)) == OK
        plans[causal] = h
    cache = RingattnPagedCache(k=x, v=x, page_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, pages=8, table_pages=4, table_stride=4, page_table=x,
                               kv_lens=x, q_starts=x, batch=2)

    def both(causal=1, tokens=0, q=x, plan=None, **scoring):
        s = RingattnPagedScoring(**dict(dict(softcap=0.0, slopes=None, prefix_lens=None, first_keys=None), **scoring))
        h = plan or plans[causal]
        a = ralib.ringattn_paged_fwd_scored(h, ctypes.byref(cache), ctypes.byref(s), q, tokens, 512, 64, x, 512, 64, x, None)
        b = ralib.ringattn_paged_weights_scored(h, ctypes.byref(cache), ctypes.byref(s), q, tokens, 512, 64, x, x, None)
        assert a == b, (a, b)
        return a

    assert both() == OK and both(softcap=30.0, slopes=x, prefix_lens=x, first_keys=x) == OK and both(causal=0, softcap=30.0) == OK
    assert both(softcap=1024.0) == OK and both(softcap=1e-6) == OK
    for bad in (float("nan"), float("inf"), -1.0, 1e-38, 3e38, 1025.0):
        assert both(softcap=bad) == E_SHAPE, bad
    for bad in ("slopes", "prefix_lens", "first_keys"):
        assert both(causal=0, **{bad: x}) == E_SHAPE and both(**{bad: x + 2}) == E_ALIGN
    assert both(plan=ctypes.c_void_p(x)) == E_PLAN and both(q=None) == E_NULL and both(tokens=65) == E_SHAPE
    assert ralib.ringattn_paged_fwd_scored(plans[1], ctypes.byref(cache), None, x, 0, 512, 64, x, 512, 64, x, None) == OK
    assert ralib.ringattn_paged_weights_scored(plans[1], None, None, x, 0, 512, 64, x, x, None) == E_NULL
    for h in plans.values():
        assert ralib.ringattn_paged_plan_destroy(h) == OK


def test_a_plan_keeps_its_scoring():
    """A cap that 32 bits do not hold is refused, not left out; what a plan was made with is not replaced under its calls."""
    memory = np.zeros(160 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    make = lambda cap: paged.PagedAttention(8, 64, kv_heads=2, page_size=16, max_batch=4, max_tokens=64, softcap=cap, workspace=(x, (160 << 20) - 16))   # noqa: E731
    for bad in (1e-50, -1e-50, -1.0, 1024.5, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            make(bad)
    plan = make(30.0)
    assert plan.softcap == 30.0 and plan.slopes is None
    with pytest.raises(AttributeError):
        plan.softcap = 50.0
    with pytest.raises(AttributeError):
        plan.slopes = torch.zeros(8)
    plan.close()
