"""The paged cache's entry points without a GPU: what they refuse, before any HIP call, and the definitions the GPU tests go by."""
import ctypes
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from ringattention_amd import _lib, paged
from ringattention_amd._lib import RingattnPagedCache, RingattnPagedParams

OK, E_NULL, E_NPES, E_DIM, E_DTYPE, E_SEQLEN, E_SHAPE, E_WS, E_RANK, E_PLAN, E_HIP, E_ALLOC, E_ALIGN = range(13)


def params(dim=64, heads=8, kv_heads=2, dtype=0, scale=0.0, page_size=16, max_batch=4, max_tokens=64, causal=1, window=0, sinks=0, flags=0):
    return RingattnPagedParams(dim, heads, kv_heads, dtype, scale, page_size, max_batch, max_tokens, causal, window, sinks, flags)


@pytest.fixture()
def memory():
    """(aligned address, bytes) of host memory that stands in for a workspace and tensors: nothing of it is touched."""
    x = np.zeros(160 << 20, dtype=np.uint8)
    base = x.ctypes.data + (-x.ctypes.data % 16)
    yield base, (160 << 20) - 16
    del x


def test_parameters(ralib, memory):
    base, size = memory

    def create(p, ws=base, n=size):
        h = ctypes.c_void_p()
        rc = ralib.ringattn_paged_plan_create(ctypes.byref(p) if p is not None else None, ctypes.c_void_p(ws), n, ctypes.byref(h))
        if rc == OK:
            assert ralib.ringattn_paged_plan_destroy(h) == OK and ralib.ringattn_paged_plan_destroy(h) == E_PLAN
        return rc

    assert create(params()) == OK and create(params(kv_heads=0)) == OK and create(params(dim=128, page_size=1024, window=5, sinks=2)) == OK
    assert create(params(causal=0, flags=1)) == OK
    assert create(None) == E_NULL
    assert ralib.ringattn_paged_plan_create(ctypes.byref(params()), None, 0, None) == E_NULL
    assert create(params(dim=96)) == E_DIM
    assert create(params(dtype=2)) == E_DTYPE
    for bad in (dict(heads=0), dict(kv_heads=3), dict(kv_heads=-1), dict(page_size=8), dict(page_size=24), dict(page_size=2048), dict(page_size=0),
                dict(max_batch=0), dict(max_batch=5000), dict(max_tokens=0), dict(max_tokens=2 ** 30), dict(window=-1), dict(sinks=-1), dict(sinks=4),
                dict(window=4, causal=0), dict(flags=2), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert create(params(**bad)) == E_SHAPE, bad
        assert ralib.ringattn_paged_workspace_bytes(ctypes.byref(params(**bad))) == 0
    need = ralib.ringattn_paged_workspace_bytes(ctypes.byref(params()))
    assert 0 < need <= size and create(params(), n=need) == OK
    assert create(params(), n=need - 1) == E_WS and create(params(), ws=base + 8) == E_ALIGN
    assert ralib.ringattn_paged_workspace_bytes(None) == 0
    assert ralib.ringattn_paged_plan_destroy(None) == E_PLAN and ralib.ringattn_paged_plan_destroy(ctypes.c_void_p(base)) == E_PLAN


def test_calls(ralib, memory):
    base, size = memory
    h = ctypes.c_void_p()
    assert ralib.ringattn_paged_plan_create(ctypes.byref(params()), ctypes.c_void_p(base), size, ctypes.byref(h)) == OK
    x = base
    good = dict(k=x, v=x, page_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, pages=8, table_pages=4, table_stride=4, page_table=x, kv_lens=x,
                q_starts=x, batch=2)

    def cache(**more):
        return ctypes.byref(RingattnPagedCache(**dict(good, **more)))

    def fwd(c, q=x, tokens=5, qt=512, qh=64, out=x, ot=512, oh=64, lse=x, plan=h):
        return ralib.ringattn_paged_fwd(plan, c, q, tokens, qt, qh, out, ot, oh, lse, None)

    def append(c, k=x, v=x, tokens=5, ts=128, hs=64, scores=None, plan=h):
        return ralib.ringattn_paged_append(plan, c, k, v, tokens, ts, hs, scores, None)

    def weights(c, q=x, tokens=5, qt=512, qh=64, lse=x, scores=x, plan=h):
        return ralib.ringattn_paged_weights(plan, c, q, tokens, qt, qh, lse, scores, None)

    def evict(c, scores=x, kept_table=x, kept_pages=2, stride=2, budget=20, first=2, last=3, kept=x, kept_lens=x, plan=h):
        return ralib.ringattn_paged_evict(plan, c, scores, kept_table, kept_pages, stride, budget, first, last, kept, kept_lens, None)

    for call in (fwd, append, weights, evict):
        assert call(cache(), plan=None) == E_PLAN and call(cache(), plan=ctypes.c_void_p(base)) == E_PLAN
        assert call(None) == E_NULL
        for bad in ("k", "page_table", "kv_lens"):
            assert call(cache(**{bad: None})) == E_NULL, bad
        for bad in (dict(batch=-1), dict(batch=5), dict(pages=0), dict(table_pages=0), dict(table_stride=3), dict(table_pages=2 ** 27, table_stride=2 ** 27),
                    dict(token_stride=32), dict(token_stride=2 ** 25), dict(token_stride=0), dict(token_stride=-64), dict(head_stride=0), dict(page_stride=0),
                    dict(page_stride=-2048), dict(page_stride=2 ** 45)):
            assert call(cache(**bad)) == E_SHAPE, bad
        for bad in (dict(k=x + 8), dict(token_stride=68), dict(head_stride=1028), dict(page_stride=2052), dict(page_table=x + 2), dict(kv_lens=x + 1)):
            assert call(cache(**bad)) == E_ALIGN, bad
        assert call(cache(batch=0)) == OK   # nothing to do
    for call in (fwd, append, evict):
        assert call(cache(v=None)) == E_NULL
    for call in (fwd, append, weights):
        assert call(cache(q_starts=None)) == E_NULL and call(cache(q_starts=x + 2)) == E_ALIGN
        assert call(cache(), tokens=-1) == E_SHAPE and call(cache(), tokens=65) == E_SHAPE
    assert fwd(cache(), tokens=0) == OK and weights(cache(v=None), tokens=0) == OK and append(cache(), tokens=0) == OK
    for bad in (dict(q=None), dict(out=None), dict(lse=None)):
        assert fwd(cache(), **bad) == E_NULL
    for bad in (dict(q=x + 8), dict(out=x + 8), dict(lse=x + 2), dict(qt=516), dict(qh=65), dict(ot=516), dict(oh=68)):
        assert fwd(cache(), **bad) == E_ALIGN, bad
    for bad in (dict(qt=-512), dict(qh=-64), dict(ot=0), dict(ot=32), dict(oh=0), dict(oh=-64), dict(qt=2 ** 40)):
        assert fwd(cache(), **bad) == E_SHAPE, bad
    for bad in (dict(k=None), dict(v=None)):
        assert append(cache(), **bad) == E_NULL
    for bad in (dict(k=x + 2), dict(v=x + 8), dict(scores=x + 1), dict(ts=130), dict(hs=60)):
        assert append(cache(), **bad) == E_ALIGN, bad
    for bad in (dict(q=None), dict(lse=None), dict(scores=None)):
        assert weights(cache(), **bad) == E_NULL
    for bad in (dict(q=x + 8), dict(lse=x + 1), dict(scores=x + 2)):
        assert weights(cache(), **bad) == E_ALIGN
    for bad in (dict(scores=None), dict(kept_table=None), dict(kept=None), dict(kept_lens=None)):
        assert evict(cache(), **bad) == E_NULL
    for bad in (dict(budget=0), dict(budget=-3), dict(first=-1), dict(last=-1), dict(first=10, last=11), dict(first=2 ** 31 - 1, last=2 ** 31 - 1)):
        assert evict(cache(), **bad) == E_SEQLEN, bad
    for bad in (dict(kept_pages=1), dict(kept_pages=0), dict(stride=1), dict(kept_pages=2 ** 27, stride=2 ** 27)):
        assert evict(cache(), **bad) == E_SHAPE, bad
    for bad in (dict(scores=x + 1), dict(kept_table=x + 2), dict(kept=x + 2), dict(kept_lens=x + 3)):
        assert evict(cache(), **bad) == E_ALIGN
    assert ralib.ringattn_paged_plan_destroy(h) == OK
    assert fwd(cache()) == E_PLAN


def test_rows_of_out_do_not_lie_on_each_other(ralib, memory):
    """Token by token or head by head, with or without room; a stride that has two rows in one place is refused before anything is launched."""
    base, size = memory
    h = ctypes.c_void_p()
    assert ralib.ringattn_paged_plan_create(ctypes.byref(params()), ctypes.c_void_p(base), size, ctypes.byref(h)) == OK
    x = base
    c = dict(k=x, v=x, page_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, pages=8, table_pages=4, table_stride=4, page_table=x, kv_lens=x,
             q_starts=x)

    def fwd(ot, oh, tokens=5, batch=0):   # (without sequences: checked, and nothing to do)
        cache = ctypes.byref(RingattnPagedCache(batch=batch, **c))
        return ralib.ringattn_paged_fwd(h, cache, x, tokens, 512, 64, x, ot, oh, x, None)

    for ot, oh in ((512, 64), (64, 320), (1024, 64), (512 + 8, 64), (64, 328), (72, 360), (1024, 128), (2 ** 36, 64), (64, 2 ** 36)):
        assert fwd(ot, oh) == OK, (ot, oh)
    for ot, oh in ((64, 64), (504, 64), (64, 312), (128, 64), (64, 128), (448, 64), (512, 72)):
        for batch in (0, 2):
            assert fwd(ot, oh, batch=batch) == E_SHAPE, (ot, oh)
    assert fwd(0, 64, tokens=1) == OK and fwd(64, 64, tokens=1) == OK
    assert ralib.ringattn_paged_plan_destroy(h) == OK


def test_tensors_that_do_not_fit(memory):
    plan = paged.PagedAttention(8, 64, kv_heads=2, page_size=16, max_batch=4, max_tokens=64, workspace=memory)
    assert plan.workspace_bytes() > 0
    half, ints = torch.float16, torch.int32
    good = dict(q=torch.zeros(5, 8, 64, dtype=half), k=torch.zeros(8, 2, 16, 64, dtype=half), v=torch.zeros(8, 2, 16, 64, dtype=half),
                table=torch.zeros(2, 4, dtype=ints), lens=torch.zeros(2, dtype=ints), starts=torch.zeros(3, dtype=ints))

    def refused(says, **more):
        x = dict(good, **more)
        with pytest.raises(ValueError, match=says):
            plan.forward(x["q"], x["k"], x["v"], x["table"], x["lens"], x["starts"])
        with pytest.raises(ValueError, match=says):
            plan.weights(x["q"], torch.zeros(8, 5), x["k"], x["table"], x["lens"], x["starts"], torch.zeros(8, 2, 16))

    refused("device tensor")   # all of it in host memory
    refused("q must be", q=torch.zeros(5, 8 * 64, dtype=half))
    refused("up to 64 new tokens", q=torch.zeros(65, 8, 64, dtype=half))
    refused("up to 4 sequences", table=torch.zeros(5, 4, dtype=ints))
    refused("kv_lens must have shape", lens=torch.zeros(3, dtype=ints))
    refused("q_starts must have shape", starts=torch.zeros(2, dtype=ints))
    refused("kv_lens must have dtype", lens=torch.zeros(2, dtype=torch.int64))
    refused("page_table must have dtype", table=torch.zeros(2, 4, dtype=torch.int64))
    refused("must be \\[pages", k=torch.zeros(8, 2, 16 * 64, dtype=half))
    def evict(says, budget, first=0, last=0, pages=2):
        with pytest.raises(ValueError, match=says):
            plan.evict(good["k"], good["v"], torch.zeros(8, 2, 16), good["table"], good["lens"], torch.zeros(2, pages, dtype=ints), budget, first, last)

    evict("device tensor", 17)
    evict("kept_table must be", 17, pages=1)
    evict("budget must be", 0)
    evict("budget must be", 8, 5, 4)
    with pytest.raises(_lib.RingattnError):
        paged.PagedAttention(8, 64, kv_heads=3, workspace=memory)
    with pytest.raises(_lib.RingattnError):
        paged.PagedAttention(8, 64, window=8, causal=False, workspace=memory)
    plan.close()
    plan.close()


def test_native_calls_leave_what_is_unusual_to_the_general_way():
    calls = _lib.load_calls()
    half = torch.float16
    for bad in ((0, 1, 0, 8, 2, 64, 16, 4, 64, 0, half, half), (1, 1, 4, 8, 2, 64, 16, 4, 64, 0, half, half), (1, 1, 0, 8, 2, 64, 16, 4, 64, 0, 1, half), (1, 1)):
        with pytest.raises((ValueError, TypeError)):
            calls.Paged(*bad)
    for kind, n in enumerate((9, 9, 8, 12)):
        call = calls.Paged(1, 1, kind, 8, 2, 64, 16, 4, 64, 0, half, half)
        for wrong in (n - 1, n + 1):
            with pytest.raises(TypeError):
                call(*(None,) * wrong)
        assert call(*(None,) * n) is None
        assert call(*(torch.zeros(1, 2, 16, 64, dtype=half),) * (n - 1), None) is None


def test_the_reference_is_plain_attention():
    """paged_reference.attend on one sequence in order against a dense softmax; the weights sum to one a row."""
    c = ref.Case("bf16", 64, 4, 2, 16, (40, 3), (40, 5), seed=1)
    out, lse, tol, _ = ref.attend(c)
    k, _ = c.rows(c.k, 0, 1)
    v, _ = c.rows(c.v, 0, 1)
    s = (c.q[:40, 2].double() @ k.T / 8).masked_fill(torch.ones(40, 40).triu(1).bool(), -math.inf)
    assert torch.allclose(out[:40, 2], torch.softmax(s, dim=1) @ v, rtol=1e-12, atol=1e-12)
    assert torch.allclose(lse[2, :40], torch.logsumexp(s, dim=1), rtol=1e-12)
    assert (out[40:42] == 0).all() and (lse[:, 40:42] == -math.inf).all()   # two new tokens of the second sequence have none to see
    clean = ref.Case("bf16", 64, 4, 2, 16, (40, 3), (40, 5), seed=1, spare=0.0)
    w, _ = ref.weights(clean, lse)
    assert abs(w.sum().item() - 4 * (40 + 3)) < 1e-9
    assert ref.kept(torch.tensor([1.0, math.nan, 3.0, 3.0, 0.0, 3.0]), torch.ones(6).bool(), 4, 1, 1) == [0, 2, 3, 5]
