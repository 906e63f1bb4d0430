"""ringattn_paged_append_rotary without a GPU: an output that has rows of K or V is refused before any HIP call."""
import ctypes

import numpy as np
import pytest

from ringattention_amd._lib import RingattnPagedCache, RingattnRotary
from test_paged import E_SHAPE, OK, params

D, HEADS, TOKENS = 64, 8, 5


@pytest.mark.parametrize("kv_heads", [1, 2, 8])
def test_an_output_on_rows_of_k_or_v_is_refused(ralib, kv_heads):
    memory = np.zeros(160 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    h = ctypes.c_void_p()
    assert ralib.ringattn_paged_plan_create(ctypes.byref(params(heads=HEADS, kv_heads=kv_heads)), ctypes.c_void_p(x), (160 << 20) - 16, ctypes.byref(h)) == OK
    cache = RingattnPagedCache(k=x, v=x, page_stride=kv_heads * 16 * D, head_stride=16 * D, token_stride=D, pages=8, table_pages=4, table_stride=4, page_table=x,
                               kv_lens=x, q_starts=x, batch=2)
    turned = RingattnRotary(D, 0, 0, 1.0, x)
    far, other = x + (1 << 20), x + (1 << 21)

    def call(q, out, k, v, qs=(HEADS * D, D), os=(HEADS * D, D), kvs=(kv_heads * D, D), tokens=TOKENS):
        return ralib.ringattn_paged_append_rotary(h, ctypes.byref(cache), ctypes.byref(turned), None, q, *qs, out, *os, k, v, tokens, *kvs, None, None)

    for tokens in (1, TOKENS):
        # in the same place, whole or from a later row on; the other of the two elsewhere
        for step in (0, D, (HEADS - 1) * D, -(kv_heads - 1) * D):
            assert call(far, other, other + 2 * step, x, tokens=tokens) == E_SHAPE, step
            assert call(far, other, x, other + 2 * step, tokens=tokens) == E_SHAPE, step
            assert call(other, other, x, other + 2 * step, tokens=tokens) == E_SHAPE, step   # in place
            assert call(other, other, other + 2 * step + 16, x, tokens=tokens) == E_SHAPE, step   # a part of a row
    # the rows of later tokens
    assert call(far, other, other + 2 * HEADS * D * 2, x, kvs=(HEADS * D, D)) == E_SHAPE
    assert call(far, other, other + 2 * (HEADS * D * 2 + 16), x, kvs=(HEADS * D, D)) == E_SHAPE
    # a fused product [tokens, (heads + 2 kv_heads) D] of which K begins a row of Q too early, or V ends in the next token's Q
    all_ = (HEADS + 2 * kv_heads) * D
    assert call(other, other, other + 2 * (HEADS - 1) * D, x, qs=(all_, D), os=(all_, D), kvs=(all_, D)) == E_SHAPE
    assert call(other, other, x, other + 2 * (all_ - (kv_heads - 1) * D - 8), qs=(all_, D), os=(all_, D), kvs=(all_, D)) == E_SHAPE
    # head by head
    assert call(far, other, other, x, os=(D, TOKENS * D), kvs=(D, TOKENS * D)) == E_SHAPE
    assert call(far, other, other + 2 * (kv_heads - 1) * TOKENS * D, x, os=(D, TOKENS * D), kvs=(D, TOKENS * D)) == E_SHAPE
    # [tokens, heads, 3, D] of which K begins within a row of Q
    if kv_heads == HEADS:
        w = 3 * D
        assert call(other, other, other + 2 * 8, x, qs=(HEADS * w, w), os=(HEADS * w, w), kvs=(HEADS * w, w)) == E_SHAPE
        assert call(other, other, x, other + 2 * (w * 4 - 8), qs=(HEADS * w, w), os=(HEADS * w, w), kvs=(HEADS * w, w)) == E_SHAPE
    assert ralib.ringattn_paged_plan_destroy(h) == OK
