"""Rotary positions without a GPU: frequencies, their form in turns, and what the entry points refuse before any HIP call."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from ringattention_amd import _lib, rotary
from ringattention_amd._lib import RingattnPagedCache, RingattnRotary, RingattnRows
from test_paged import params

OK, E_NULL, E_NPES, E_DIM, E_DTYPE, E_SEQLEN, E_SHAPE, E_WS, E_RANK, E_PLAN, E_HIP, E_ALLOC, E_ALIGN = range(13)
TWO_PI = Fraction("6.28318530717958647692528676655900576839433879875021164194988918461563281257241799725606965068423413596")


def turns(lib, radians):
    made = (ctypes.c_uint64 * max(1, len(radians)))()
    rc = lib.ringattn_rotary_turns((ctypes.c_double * max(1, len(radians)))(*radians), len(radians), made)
    return rc, [int(x) for x in made][:len(radians)]


def test_turns(ralib):
    radians = [1.0, 1e-4, 0.123456789, 0.0, 6.28, 100.0, -0.5, -1e-30, 2.0 ** -70]
    rc, made = turns(ralib, radians)
    assert rc == OK
    for x, t in zip(radians, made):
        want = (Fraction(x) / TWO_PI % 1) * 2 ** 64
        off = abs(Fraction(t) - want)
        off = min(off, 2 ** 64 - off)
        # 64-bit significands: the quotient, its whole turns, and the rounding to an integer
        assert off <= 1 + max(abs(x) / 6.28, 1) * 2.0 ** 64 * 2.0 ** -62, (x, float(off))
    assert turns(ralib, [float("inf")])[0] == E_SHAPE and turns(ralib, [1.0, float("nan")])[0] == E_SHAPE
    assert turns(ralib, [])[0] == OK
    assert ralib.ringattn_rotary_turns(None, 1, (ctypes.c_uint64 * 1)()) == E_NULL and ralib.ringattn_rotary_turns((ctypes.c_double * 1)(), 1, None) == E_NULL
    assert ralib.ringattn_rotary_turns((ctypes.c_double * 1)(), -1, (ctypes.c_uint64 * 1)()) == E_SHAPE


def test_frequencies():
    plain, scale = rotary.frequencies(128)
    assert scale == 1 and plain == [10000.0 ** (-i / 64) for i in range(64)]
    linear, _ = rotary.frequencies(128, scaling="linear", factor=4)
    assert linear == [x / 4 for x in plain]
    ntk, _ = rotary.frequencies(128, scaling="ntk", factor=8)
    assert ntk[0] == 1 and math.isclose(ntk[-1], plain[-1] / 8, rel_tol=1e-12) and all(a >= b for a, b in zip(plain, ntk))
    yarn, scale = rotary.frequencies(128, scaling="yarn", factor=16, trained=4096)
    assert math.isclose(scale, 0.1 * math.log(16) + 1)
    assert yarn[0] == plain[0] and math.isclose(yarn[-1], plain[-1] / 16)
    for i, (x, y) in enumerate(zip(plain, yarn)):
        if 4096 * x / (2 * math.pi) > 34:
            assert y == x
        if 4096 * x / (2 * math.pi) < 0.9:
            assert math.isclose(y, x / 16)
        assert x / 16 * (1 - 1e-12) <= y <= x
    assert rotary.frequencies(16, scaling="ntk", factor=2)[0][0] == 1
    assert rotary.frequencies(2, scaling="ntk", factor=2)[0] == [1.0]
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=16, base=1), dict(rotary_dim=16, base=float("nan")), dict(rotary_dim=16, scaling="other"),
                dict(rotary_dim=16, factor=2), dict(rotary_dim=16, scaling="linear", factor=0.5), dict(rotary_dim=16, scaling="yarn", factor=2),
                dict(rotary_dim=16, scaling="linear", factor=float("inf"))):
        with pytest.raises(ValueError):
            rotary.frequencies(**bad)


def test_rotary_parameters(ralib):
    r = rotary.Rotary(128, 64, interleaved=True, dtype="bf16", device="cpu")
    assert r.turns.shape == (32,) and r.params(True).inverse == 1 and r.params(False).inverse == 0
    assert rotary.Rotary(64, radians=[0.1] * 32, scale=2.0, device="cpu").scale == 2
    for bad in (dict(dim=96), dict(dim=64, rotary_dim=128), dict(dim=64, rotary_dim=24), dict(dim=64, rotary_dim=8), dict(dim=64, rotary_dim=-16),
                dict(dim=64, radians=[1.0]), dict(dim=64, radians=[float("nan")] * 32), dict(dim=64, radians=[1.0] * 32, scaling="linear", factor=2.0),
                dict(dim=64, scale=0.0), dict(dim=64, scale=float("inf")), dict(dim=64, scale=-1.0), dict(dim=64, scale=1e-60)):
        with pytest.raises(ValueError):
            rotary.Rotary(device="cpu", **bad)
    with pytest.raises(KeyError):
        rotary.Rotary(64, dtype="fp32", device="cpu")
    x = torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        r.apply(x)
    for bad in (x[0], x[..., :64], x.half(), x[None, None]):
        with pytest.raises(ValueError):
            r.apply(bad)


def test_apply_refusals(ralib):
    memory = np.zeros(1 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    turned = dict(rotary_dim=64, interleaved=0, inverse=0, factor=0.0, turns=x)
    tensor = dict(in_=x, out=x, heads=2, in_batch_stride=0, in_head_stride=64, in_token_stride=128, out_batch_stride=0, out_head_stride=64, out_token_stride=128)

    def call(dim=64, dtype=0, count=1, batch=1, tokens=3, positions=None, stride=0, second=None, rotary=turned, **more):
        rows = (RingattnRows * 2)(RingattnRows(**dict(tensor, **more)), RingattnRows(**dict(tensor, **(second or {}))))
        r = RingattnRotary(**rotary) if rotary else None
        return ralib.ringattn_rotary_apply(ctypes.byref(r) if r else None, dim, dtype, rows if count else None, count or 1, batch, tokens, positions, stride, None)

    assert call(dim=96) == E_DIM and call(dtype=2) == E_DTYPE and call(rotary=None) == E_NULL and call(count=0) == E_NULL
    for bad, code in ((dict(turns=None), E_NULL), (dict(turns=x + 4), E_ALIGN), (dict(rotary_dim=0), E_DIM), (dict(rotary_dim=128), E_DIM), (dict(rotary_dim=24), E_DIM),
                      (dict(factor=float("nan")), E_SHAPE), (dict(factor=-1.0), E_SHAPE), (dict(factor=float("inf")), E_SHAPE)):
        assert call(rotary=dict(turned, **bad)) == code, bad
    far = x + (1 << 19)
    for bad, code in ((dict(count=3), E_SHAPE), (dict(batch=-1), E_SHAPE), (dict(batch=65536), E_SHAPE), (dict(tokens=-1), E_SHAPE), (dict(tokens=2 ** 30 + 1), E_SHAPE),
                      (dict(positions=x + 2), E_ALIGN), (dict(positions=x, stride=-1), E_SHAPE), (dict(in_=None), E_NULL), (dict(out=None), E_NULL),
                      (dict(heads=0), E_SHAPE), (dict(heads=65536), E_SHAPE), (dict(in_=x + 8), E_ALIGN), (dict(out=x + 8), E_ALIGN),
                      (dict(in_head_stride=60), E_ALIGN), (dict(out_token_stride=132), E_ALIGN), (dict(in_token_stride=-128), E_SHAPE),
                      (dict(in_token_stride=2 ** 37), E_SHAPE), (dict(out=far, out_head_stride=32), E_SHAPE), (dict(out=far, out_token_stride=64), E_SHAPE),
                      (dict(out=far, out_head_stride=0), E_SHAPE), (dict(batch=2, out=far, out_batch_stride=64), E_SHAPE), (dict(out=far, batch=2), E_SHAPE),
                      (dict(out=x + 64 * 2), E_SHAPE), (dict(out_token_stride=256), E_SHAPE), (dict(count=2, second=dict(heads=0)), E_SHAPE), (dict(heads=40000, tokens=0, count=2, second=dict(heads=40000)), E_SHAPE),
                      (dict(count=2, second=dict(out=x + 256)), E_SHAPE)):
        assert call(**bad) == code, bad
    # nothing to do is no error, and strides of dimensions of one entry count for nothing
    assert call(tokens=0) == OK and call(batch=0) == OK
    assert call(tokens=0, heads=1, in_head_stride=3) == OK


def test_outputs_in_the_other_tensor_are_refused(ralib):
    memory = np.zeros(1 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    far, further = x + (1 << 18), x + (1 << 19)
    r = RingattnRotary(64, 0, 0, 1.0, x)

    def call(first, second):
        rows = (RingattnRows * 2)(*(RingattnRows(i, o, 2, 2 * 5 * 64, 5 * 64, 64, 2 * 5 * 64, 5 * 64, 64) for i, o in (first, second)))
        return ralib.ringattn_rotary_apply(ctypes.byref(r), 64, 0, rows, 2, 1, 5, None, 0, None)

    assert call((x, far), (further, far)) == E_SHAPE        # one output for both
    assert call((x, far), (far, further)) == E_SHAPE        # Q turned over K
    assert call((x, far), (further, x)) == E_SHAPE          # K turned over Q
    assert call((x, x), (x, x)) == E_SHAPE and call((x, x), (x, far)) == E_SHAPE


def test_append_rotary_refusals(ralib):
    memory = np.zeros(160 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    h = ctypes.c_void_p()
    assert ralib.ringattn_paged_plan_create(ctypes.byref(params()), ctypes.c_void_p(x), (160 << 20) - 16, ctypes.byref(h)) == OK
    cache = dict(k=x, v=x, page_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, pages=8, table_pages=4, table_stride=4, page_table=x, kv_lens=x,
                 q_starts=x, batch=2)
    turned = dict(rotary_dim=64, interleaved=0, inverse=0, factor=1.0, turns=x)
    far = x + (1 << 20)

    def call(plan=h, c=None, r=None, positions=None, q=x, qt=512, qh=64, out=far, ot=512, oh=64, k=x, v=x, tokens=5, ts=128, hs=64, scores=None):
        c, r = RingattnPagedCache(**dict(cache, **(c or {}))), RingattnRotary(**dict(turned, **(r or {})))
        return ralib.ringattn_paged_append_rotary(plan, ctypes.byref(c), ctypes.byref(r), positions, q, qt, qh, out, ot, oh, k, v, tokens, ts, hs, scores, None)

    for bad, code in ((dict(plan=None), E_PLAN), (dict(c=dict(k=None)), E_NULL), (dict(c=dict(batch=5)), E_SHAPE), (dict(c=dict(q_starts=None)), E_NULL),
                      (dict(r=dict(turns=None)), E_NULL), (dict(r=dict(rotary_dim=72)), E_DIM), (dict(r=dict(rotary_dim=128)), E_DIM), (dict(q=None), E_NULL),
                      (dict(out=None), E_NULL), (dict(k=None), E_NULL), (dict(v=None), E_NULL), (dict(tokens=65), E_SHAPE), (dict(tokens=-1), E_SHAPE),
                      (dict(qt=516), E_ALIGN), (dict(oh=60), E_ALIGN), (dict(oh=32), E_SHAPE), (dict(ts=129), E_ALIGN), (dict(hs=-8), E_SHAPE), (dict(q=x + 8), E_ALIGN),
                      (dict(out=far + 8), E_ALIGN), (dict(k=x + 2), E_ALIGN), (dict(positions=x + 1), E_ALIGN), (dict(scores=x + 2), E_ALIGN),
                      (dict(out=x + 512), E_SHAPE), (dict(out=x, ot=1024), E_SHAPE)):
        assert call(**bad) == code, bad
    assert call(tokens=0) == OK and call(c=dict(batch=0)) == OK
    assert ralib.ringattn_paged_plan_destroy(h) == OK


def test_native_calls_leave_what_is_unusual_to_the_general_way(ralib):
    """Rotary positions, pages, and the paged calls with scores that are shaped or rows that turn (csrc/ringattn_calls.cpp): what is no device tensor of the
    expected kind gives None, a wrong number of arguments is refused."""
    from ringattention_amd import paged
    calls = _lib.load_calls()
    half = torch.float16
    x = torch.zeros(1, 2, 16, 64, dtype=half)
    r = rotary.Rotary(64, device="cpu")
    for kind, n in ((16, 12), (17, 11), (18, 14)):
        call = calls.Paged(1, 1, kind, 8, 2, 64, 16, 4, 64, 0, half, half, 30.0)
        for wrong in (n - 1, n + 1):
            with pytest.raises(TypeError):
                call(*(None,) * wrong)
        assert call(*(None,) * n) is None and call(*(x,) * (n - 1), None) is None
    for bad in (19, 15, -1):
        with pytest.raises(ValueError):
            calls.Paged(1, 1, bad, 8, 2, 64, 16, 4, 64, 0, half, half)
    turn = calls.Turn(1, r.address, r.address, 64, 0, 0, half)
    pool = paged.PagePool(1, 2, 3, 16, device="cpu")
    pages = calls.Pages(1, ctypes.addressof(pool._struct), 0, 0)
    for call in (turn, pages):
        for wrong in (6, 8):
            with pytest.raises(TypeError):
                call(*(None,) * wrong)
        assert call(*(None,) * 7) is None and call(x, x, None, None, None, x, None) is None and call(*(x,) * 6, None) is None
    for make, bad in ((calls.Turn, (0, 1, 1, 64, 0, 0, half)), (calls.Turn, (1, 0, 1, 64, 0, 0, half)), (calls.Turn, (1, 1, 1, 64, 0, 0, 1)), (calls.Turn, (1,)),
                      (calls.Pages, (1, 1, 2, 0)), (calls.Pages, (0, 1, 0, 0)), (calls.Pages, (1, 0, 0, 0)), (calls.Pages, (1, 1))):
        with pytest.raises((ValueError, TypeError)):
            make(*bad)
