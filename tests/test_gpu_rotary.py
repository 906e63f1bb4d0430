"""Rotary positions on the GPU against the definition in 64 bits.

How far a column may be off: half a step of the storage type of what it is; and in 32 bits an angle that is off by 2^-26 of a turn (2^-23.3
radians), a sine and a cosine that are off by 2^-21, the factor's and two products' and a sum's roundings of 2^-24 each -- altogether less than
2^-19.5 of |x_a| + |x_b| times the factor.  fp16 below its normal range: half its smallest step."""
import math
from fractions import Fraction

import pytest
import torch

import paged_reference as ref
from ringattention_amd import api, paged
from ringattention_amd.rotary import Rotary
from test_rotary import TWO_PI

pytestmark = pytest.mark.gpu


def angles(rotary, positions):
    """Angles [..., pairs] in 64 bits, from whole numbers: exact for any position."""
    out = []
    for p in positions.reshape(-1).tolist():
        out.append([float(Fraction(p) * Fraction(f) / TWO_PI % 1) * 2 * math.pi for f in rotary.radians])
    return torch.tensor(out, dtype=torch.float64).reshape(*positions.shape, len(rotary.radians))


def expected(rotary, x, ang, inverse=False):
    """(y, how far off) for x [..., dim] and angles [..., pairs] that go with it."""
    x, r = x.double().cpu(), rotary.rotary_dim
    t = x[..., :r]
    a, b = (t[..., 0::2], t[..., 1::2]) if rotary.interleaved else (t[..., :r // 2], t[..., r // 2:])
    c, s = torch.cos(ang), torch.sin(ang) * (-1 if inverse else 1)
    p, q, size = rotary.scale * (a * c - b * s), rotary.scale * (b * c + a * s), rotary.scale * (a.abs() + b.abs())
    def join(p, q):   # noqa: E306
        return torch.stack((p, q), dim=-1).flatten(-2) if rotary.interleaved else torch.cat((p, q), dim=-1)
    y = torch.cat((join(p, q), x[..., r:]), dim=-1)
    size = torch.cat((join(size, size), torch.zeros_like(x[..., r:])), dim=-1)
    u = 2.0 ** -8 if rotary.torch_dtype == torch.bfloat16 else 2.0 ** -11
    tol = u * (y.abs() + 2.0 ** -19.5 * size) + 2.0 ** -19.5 * size + (2.0 ** -25 if u < 2.0 ** -8 else 0.0)
    tol[..., r:] = 0   # columns that stay are copied
    return y, tol


def close(got, want, tol):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), ((got - want).abs() - tol)[bad].max())


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (64, 16), (64, 48), (128, 128), (128, 32), (128, 112)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 3, 70])
def test_forms(dtype, dim, rotary_dim, interleaved, tokens):
    r = Rotary(dim, rotary_dim, interleaved=interleaved, scaling="yarn", factor=4, trained=64, dtype=dtype)
    q, k = normal((2, 5, tokens, dim), r.torch_dtype, 1), normal((2, 2, tokens, dim), r.torch_dtype, 2)
    ang = angles(r, torch.arange(tokens))
    qo, ko = r.apply(q, k)
    close(qo, *expected(r, q, ang))
    close(ko, *expected(r, k, ang))
    # back, in place, tokens first
    t = q.transpose(1, 2)[1].clone()
    pos = torch.tensor([(7919 * i) % 1000 - 300 for i in range(tokens)], dtype=torch.int32)
    want = expected(r, t, angles(r, pos)[:, None], inverse=True)
    got, none = r.apply(t, positions=pos.cuda(), q_out=t, inverse=True)
    assert none is None and got.data_ptr() == t.data_ptr()
    close(t, *want)


def test_far_positions():
    r = Rotary(128, dtype="fp16", base=500000.0)
    pos = torch.tensor([0, 1, 2 ** 20 + 1, 10 ** 8 + 7, 2 ** 30 - 1, 2 ** 31 - 1, -1, -2 ** 31, -123456789], dtype=torch.int32)
    q = normal((len(pos), 3, 128), torch.float16, 3)
    got, _ = r.apply(q, positions=pos.cuda())
    close(got, *expected(r, q, angles(r, pos)[:, None]))


def test_gradient_against_differences():
    """The inverse with the forward's factor is the forward's transpose: <g, R x> = <R' g, x>, and by differences along single columns."""
    r = Rotary(64, 32, interleaved=True, scaling="yarn", factor=8, trained=128, dtype="fp16")
    g, x = normal((1, 2, 9, 64), torch.float16, 4), normal((1, 2, 9, 64), torch.float16, 5)
    back = r.apply(g, inverse=True)[0].double().cpu()
    ang = angles(r, torch.arange(9))
    for column in (0, 1, 17, 31, 32, 63):
        e = torch.zeros_like(x)
        e[..., column] = 1
        # the map is linear, so that a difference over any step is its derivative: exact but for the roundings of its two sides
        up, down = r.apply(x + e)[0].double().cpu(), r.apply(x)[0].double().cpu()
        step = (x + e).double().cpu()[..., column] - x.double().cpu()[..., column]
        slope = ((up - down) * g.double().cpu()).sum(-1)
        size = (expected(r, x + e, ang)[1] + expected(r, x, ang)[1]) * g.double().cpu().abs()
        tol = size.sum(-1) + expected(r, g, ang, True)[1][..., column] * step.abs() + 1e-9
        assert ((slope - back[..., column] * step).abs() <= tol).all(), column


def test_layouts_and_streams():
    r = Rotary(128, dtype="bf16")
    base = normal((2, 40, 12, 128), torch.bfloat16, 6)    # a fused projection: [batch, tokens, heads of q, k, v, dim]
    q, k = base[:, :, :8].transpose(1, 2), base[:, :, 8:10].transpose(1, 2)
    pos = torch.stack([torch.arange(40), torch.arange(40) * 3 + 5]).int()
    ang = angles(r, pos)[:, None]
    want_q, want_k, rest = expected(r, q, ang), expected(r, k, ang), base[:, :, 10:].clone()
    qo, ko = r.apply(q, k, pos.cuda())
    close(qo, *want_q)
    close(ko, *want_k)
    assert qo.stride() == torch.empty_like(q).stride()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    r.apply(q, k, pos.cuda(), q_out=q, k_out=k, stream=stream)
    stream.synchronize()
    close(q, *want_q)
    close(k, *want_k)
    assert torch.equal(base[:, :, 10:], rest)
    # tensors of no tokens, no batch
    for shape in ((0, 4, 3, 128), (1, 4, 0, 128), (0, 4, 128)):
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        assert r.apply(x, x)[1].shape == shape


def test_zigzag_positions():
    r = Rotary(64, dtype="fp16")
    order = torch.from_numpy(api.zigzag_order([8, 8, 8, 8]))
    x = normal((1, 2, 32, 64), torch.float16, 7)
    whole = r.apply(x)[0]
    dealt = r.apply(x[:, :, order.cuda()].contiguous(), positions=order.int().cuda())[0]
    assert torch.equal(dealt, whole[:, :, order.cuda()])


def test_refusals():
    r = Rotary(64, dtype="fp16")
    x = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    wide = torch.zeros(4, 2, 72, dtype=torch.float16, device="cuda")
    for call in (lambda: r.apply(wide[..., 4:68]), lambda: r.apply(x, x[:3]), lambda: r.apply(x, x[None]), lambda: r.apply(x, k_out=x), lambda: r.apply(x.cpu()),
                 lambda: r.apply(x, positions=torch.arange(4, device="cuda")), lambda: r.apply(x, positions=torch.arange(3, device="cuda").int()),
                 lambda: r.apply(x, positions=torch.zeros(1, 4, device="cuda").int()), lambda: r.apply(x, q_out=x[:2]), lambda: r.apply(x, q_out=x.float()),
                 lambda: Rotary(64, dtype="fp16", device="cpu").apply(x)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):   # rows on each other
        r.apply(x, q_out=x[:1].expand(4, 2, 64))
    both = torch.zeros(8, 2, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError):   # neither the tensor itself nor elsewhere
        r.apply(both[:4], q_out=both[2:6])


# ---- into the paged cache

def state(c):
    return {k: getattr(c, k).cuda() for k in ("q", "k", "v", "table", "starts")} | {"lens": c.kv_lens().cuda()}


def places(c):
    """(sequence, position) of every new token that a sequence has."""
    return [(b, c.lens[b] - c.news[b] + i) for b in range(len(c.lens)) for i in range(c.news[b])]


CASES = [dict(lens=[5], news=[1]), dict(lens=[1], news=[1], dim=64), dict(lens=[40, 17, 3, 64], news=[7, 1, 3, 0], dtype="fp16", dim=64, extra_rows=3),
         dict(lens=[100, 33], news=[100, 2], heads=8, kv_heads=1, page=32), dict(lens=list(range(1, 71)), news=[1] * 70, heads=2, kv_heads=2),
         dict(lens=[2, 9], news=[5, 1], extra_rows=1), dict(lens=[129], news=[129], heads=3, kv_heads=3, dim=64)]


@pytest.mark.parametrize("n", range(len(CASES)))
@pytest.mark.parametrize("how", ["", "positions", "in place", "head major"])
def test_append(n, how):
    c = ref.Case(**CASES[n], seed=n, spare=7.0)
    s = state(c)
    r = Rotary(c.dim, c.dim // 2 if n % 2 else 0, interleaved=n % 3 == 0, scaling="linear", factor=2, dtype=c.dtype)
    plan = paged.PagedAttention(c.heads, c.dim, kv_heads=c.kv_heads, dtype=c.dtype, page_size=c.page, max_batch=len(c.lens), max_tokens=c.tokens)
    k, v = (normal((c.tokens, c.kv_heads, c.dim), r.torch_dtype, 20 + i) for i in range(2))
    q, q_out = s["q"], None
    pos = torch.tensor([(31 * i) % 501 - 40 for i in range(c.tokens)], dtype=torch.int32) if how == "positions" else None
    if how == "in place":
        q_out = q
    elif how == "head major":
        q = s["q"].transpose(0, 1).contiguous().transpose(0, 1)
        k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
        q_out = torch.full((c.heads, c.tokens, c.dim), 5.0, dtype=r.torch_dtype, device="cuda").transpose(0, 1)
    else:
        q_out = torch.full_like(q, 5.0)
    there = places(c)
    T = len(there)
    at = pos[:T] if pos is not None else torch.tensor([p for _, p in there], dtype=torch.int32)
    ang = angles(r, at)[:, None]
    want_q, want_k = expected(r, q[:T], ang), expected(r, k[:T], ang)
    behind = q_out[T:].clone()
    k_cache, v_cache = c.k.clone().cuda(), c.v.clone().cuda()
    scores = torch.ones(c.pages, c.kv_heads, c.page, device="cuda")
    got = plan.append_rotary(r, q, k, v, k_cache, v_cache, s["table"], s["lens"], s["starts"], scores, pos.cuda() if pos is not None else None, q_out)
    assert got is q_out
    close(q_out[:T], *want_q)
    assert torch.equal(q_out[T:], behind)
    k_want, v_want, s_want = c.k.double(), c.v.clone(), torch.ones(c.pages, c.kv_heads, c.page)
    tol = torch.zeros_like(k_want)
    for t, (b, p) in enumerate(there):
        page = c.row(b, p) if p >= 0 else None
        if page is not None:
            k_want[page, :, p % c.page], tol[page, :, p % c.page] = want_k[0][t], want_k[1][t]
            v_want[page, :, p % c.page] = v[t].cpu()
            s_want[page, :, p % c.page] = 0
    close(k_cache, k_want, tol)
    assert torch.equal(v_cache.cpu(), v_want) and torch.equal(scores.cpu(), s_want)


def test_append_is_apply_and_append():
    """The same bits as turning Q and K first and appending then, also of a captured call whose lengths change between replays."""
    c = ref.Case(lens=[40, 17, 3, 64], news=[7, 1, 3, 2], seed=3, spare=0.0)
    s = state(c)
    r = Rotary(c.dim, dtype=c.dtype)
    plan = paged.PagedAttention(c.heads, c.dim, kv_heads=c.kv_heads, dtype=c.dtype, page_size=c.page, max_batch=4, max_tokens=c.tokens)
    k, v = (normal((c.tokens, c.kv_heads, c.dim), r.torch_dtype, 30 + i) for i in range(2))
    q_out, kc, vc = torch.empty_like(s["q"]), c.k.cuda(), c.v.cuda()
    seqs = (s["table"], s["lens"], s["starts"])
    plan.append_rotary(r, s["q"], k, v, kc, vc, *seqs, q_out=q_out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.append_rotary(r, s["q"], k, v, kc, vc, *seqs, q_out=q_out)
    for shift in (0, 1, 2):
        lens = [x + shift if x != 64 else x for x in c.lens]
        s["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        kc.copy_(c.k)
        vc.copy_(c.v)
        graph.replay()
        pos = torch.tensor([lens[b] - c.news[b] + i for b in range(4) for i in range(c.news[b])], dtype=torch.int32).cuda()
        k2, v2 = c.k.cuda(), c.v.cuda()
        q_turned, k_turned = r.apply(s["q"], k, pos)
        plan.append(k_turned, v, k2, v2, *seqs)
        torch.cuda.synchronize()
        assert torch.equal(q_turned, q_out) and torch.equal(kc, k2) and torch.equal(vc, v2), shift


def test_append_pages_that_are_not_there_and_odd_starts():
    """Guard rows around everything that is written, entries outside the pool, lengths and starts of any kind."""
    c = ref.Case(lens=[40, 17, 30], news=[9, 4, 2], seed=5, spare=0.0, extra_rows=2)
    r = Rotary(c.dim, dtype=c.dtype)
    plan = paged.PagedAttention(c.heads, c.dim, kv_heads=c.kv_heads, dtype=c.dtype, page_size=c.page, max_batch=3, max_tokens=c.tokens)
    k, v = (normal((c.tokens, c.kv_heads, c.dim), r.torch_dtype, 40 + i) for i in range(2))
    for table_fix, lens, starts in (({(0, 2): -1, (1, 1): 99}, c.lens, None), ({}, [2 ** 31 - 1, -5, 0], None), ({}, c.lens, [5, 2, 17, 3]), ({}, c.lens, [-7, 3, 40, 2 ** 31 - 1])):
        table = c.table.clone()
        for at, e in table_fix.items():
            table[at] = e
        big_q = torch.full((c.tokens + 2, c.heads, c.dim), 3.0, dtype=r.torch_dtype, device="cuda")
        big = [torch.full((c.pages + 2, c.kv_heads, c.page, c.dim), 3.0, dtype=r.torch_dtype, device="cuda") for _ in range(2)]
        st = c.starts if starts is None else torch.tensor(starts, dtype=torch.int32)
        plan.append_rotary(r, c.q.cuda(), k, v, big[0][1:-1], big[1][1:-1], table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), st.cuda(), q_out=big_q[1:-1])
        torch.cuda.synchronize()
        for x in big + [big_q]:
            assert (x[0] == 3).all() and (x[-1] == 3).all()
        if table_fix:   # the rows of Q are there all the same; nothing lands on page 0 or elsewhere
            ang = angles(r, torch.tensor([p for _, p in places(c)]))[:, None]
            close(big_q[1:1 + 15], *expected(r, c.q[:15], ang))
            written = {(c.row(b, p), p % c.page) for b, p in places(c) if (b, p // c.page) not in table_fix}
            touched = (big[1][1:-1] != 3).any(dim=3).any(dim=1).cpu()
            assert {(i, j) for i in range(c.pages) for j in range(c.page) if touched[i, j]} <= written


def test_offsets_past_32_bits():
    """Rows behind the first 2^32 elements, and pages behind them: the same bits as near the beginning."""
    r = Rotary(64, dtype="bf16")
    n = 2 ** 26 + 5
    x = torch.empty(n, 1, 64, dtype=torch.bfloat16, device="cuda")
    x[-70:] = normal((70, 1, 64), torch.bfloat16, 50)
    last, want = x[-70:].clone(), torch.arange(n - 70, n, dtype=torch.int32).cuda()
    got = r.apply(last, positions=want)[0]
    r.apply(x, q_out=x)
    assert torch.equal(x[-70:], got)
    del x
    c = ref.Case(lens=[40], news=[40], heads=2, kv_heads=1, dim=64, seed=9)
    pages = 2 ** 22 + 3    # of 16 x 64
    k_cache, v_cache = (torch.zeros(pages, 1, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k, v = (normal((40, 1, 64), torch.bfloat16, 51 + i) for i in range(2))
    plan = paged.PagedAttention(2, 64, kv_heads=1, dtype="bf16", page_size=16, max_batch=1, max_tokens=40)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32).cuda()
    lens, starts = torch.tensor([40], dtype=torch.int32).cuda(), torch.tensor([0, 40], dtype=torch.int32).cuda()
    plan.append_rotary(r, c.q.cuda(), k, v, k_cache, v_cache, table, lens, starts)
    want = r.apply(k)[0]
    at = torch.cat([torch.arange(16) + 16 * p for p in table[0].tolist()])[:40].cuda()
    assert torch.equal(k_cache.view(-1, 64)[at], want[:, 0]) and torch.equal(v_cache.view(-1, 64)[at], v[:, 0])
    assert not k_cache[:-3].any() and not v_cache[:-3].any()
