"""Capped, sloped and masked scores over the paged cache on the GPU, against the definition in 64 bits (scored_reference)."""
import math

import pytest
import torch

import scored_reference as ref
from ringattention_amd import api, paged

pytestmark = pytest.mark.gpu


def plan_of(c, **more):
    return paged.PagedAttention(c.heads, c.dim, kv_heads=c.kv_heads, dtype=c.dtype, page_size=c.page, max_batch=max(1, len(c.lens)), max_tokens=max(1, c.tokens),
                                causal=c.causal, window=c.window, sinks=c.sinks, softcap=c.cap, slopes=c.given()[0], **more)


def sequences(c):
    return c.table.cuda(), c.kv_lens().cuda(), c.starts.cuda()


def compare(got, want, tol, what):
    got, want = got.double().cpu(), want
    same = (got == want) | (got.isnan() & want.isnan()) | ((got - want).abs() <= tol)
    assert same.all(), (what, int((~same).sum()), got[~same][:4], want[~same][:4], tol[~same][:4])


def check(c, do_weights=True, **more):
    plan = plan_of(c, **more)
    slopes, prefix, first = c.given()
    q, k, v = c.q.cuda(), c.k.cuda(), c.v.cuda()
    out = torch.full((c.tokens, c.heads, c.dim), 5.0, dtype=q.dtype, device="cuda")
    lse = torch.full((c.heads, c.tokens), 5.0, device="cuda")
    plan.forward(q, k, v, *sequences(c), out, lse, prefix_lens=prefix, first_keys=first)
    want, want_lse, tol, tol_lse = ref.attend(c)
    T = int(c.starts[-1])
    assert (out[T:] == 5).all() and (lse[:, T:] == 5).all()
    compare(out[:T], want[:T], tol[:T], "out")
    compare(lse[:, :T], want_lse[:, :T], tol_lse[:, :T], "lse")
    if do_weights:
        scores = torch.zeros(c.pages, c.kv_heads, c.page, device="cuda")
        plan.weights(q, lse, k, *sequences(c), scores, prefix_lens=prefix, first_keys=first)
        compare(scores, *ref.weights(c, lse.cpu()), "weights")
    return out, lse


def slopes_of(heads):
    return [2.0 ** (-8 * (h + 1) / heads) for h in range(heads)]


def docs_of(c_lens, news, size):
    return [(L - n + i) // size * size for L, n in zip(c_lens, news) for i in range(n)]


BATCHES = {
    "one": dict(lens=[1], news=[1], heads=2, kv_heads=1),
    "tokens": dict(lens=[65, 1, 300, 47, 129], news=[1, 1, 1, 1, 1], heads=8, kv_heads=2),
    "few": dict(lens=[70, 33, 200], news=[9, 33, 2], heads=4, kv_heads=4, page=32),
    "many": dict(lens=[700, 90], news=[531, 90], heads=4, kv_heads=2, page=64),
    "mixed": dict(lens=[400, 1, 0, 260, 31], news=[300, 1, 0, 1, 3], heads=6, kv_heads=2, extra_rows=2),
    "more new than there": dict(lens=[3, 40], news=[9, 5], heads=2, kv_heads=2),
}
SCORES = {
    "cap": lambda b: dict(cap=3.0),
    "slopes": lambda b: dict(slopes=slopes_of(b["heads"])),
    "cap and slopes": lambda b: dict(cap=50.0, slopes=slopes_of(b["heads"])),
    "prefix": lambda b: dict(prefix=[(37 * i + 50) % 131 for i in range(len(b["lens"]))]),
    "documents": lambda b: dict(first=docs_of(b["lens"], b["news"], 29) + [0] * b.get("extra_rows", 0)),
    "all": lambda b: dict(cap=5.0, slopes=slopes_of(b["heads"]), prefix=[(i * 7) % 20 for i in range(len(b["lens"]))], window=60, sinks=3,
                          first=docs_of(b["lens"], b["news"], 43) + [0] * b.get("extra_rows", 0)),
    "window and prefix": lambda b: dict(prefix=[11] * len(b["lens"]), window=33, sinks=2, slopes=slopes_of(b["heads"])),
}


@pytest.mark.parametrize("scores", SCORES)
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("fp16", 64)])
def test_against_the_definition(batch, scores, dtype, dim):
    b = BATCHES[batch]
    check(ref.Case(**SCORES[scores](b), **b, dtype=dtype, dim=dim, sigma=1.5, seed=len(batch) + len(scores)))


@pytest.mark.parametrize("dtype,dim", [("fp16", 128), ("bf16", 64)])
def test_the_other_types(dtype, dim):
    for name in ("mixed", "many"):
        b = BATCHES[name]
        for scores in ("cap and slopes", "all"):
            check(ref.Case(**SCORES[scores](b), **b, dtype=dtype, dim=dim, sigma=1.5, seed=9))


@pytest.mark.parametrize("cap", [1e-3, 0.5, 200.0, 1024.0])
def test_caps_small_and_large(cap):
    for b in ("tokens", "many"):
        check(ref.Case(cap=cap, **BATCHES[b], dtype="fp16", dim=64, sigma=3.0, seed=11))


def test_slopes_of_either_sign():
    """And of a size at which a few keys are all that counts."""
    for b in ("few", "many"):
        check(ref.Case(slopes=[-0.25, 8.0, 0.0, -1e-3], **dict(BATCHES[b], heads=4), seed=13))
        check(ref.Case(slopes=[-0.25, 8.0, 0.0, -1e-3], prefix=[40] * len(BATCHES[b]["lens"]), **dict(BATCHES[b], heads=4), seed=14))


@pytest.mark.parametrize("n", range(6))
def test_first_keys_of_any_kind(n):
    """Out of order, negative, behind the token itself (which then sees nothing but a prefix), behind the end."""
    g = torch.Generator().manual_seed(n)
    lens, news = ([500, 77], [290, 9]) if n % 2 else ([900, 40, 20], [1, 7, 20])
    first = [int(x) for x in torch.randint(-50, 1000, (sum(news),), generator=g)]
    if n < 2:
        first = [2 ** 31 - 1 if x > 500 else x for x in first]
    more = [{}, dict(prefix=[5, 0, 30][:len(lens)]), dict(window=70, sinks=4)][n // 2]
    out, lse = check(ref.Case(lens=lens, news=news, heads=4, kv_heads=2, first=first, seed=n, **more))
    if n < 2:
        assert (lse == -math.inf).any() and torch.isfinite(out).all()


@pytest.mark.parametrize("prefix", [[0, 0], [-5, 2 ** 31 - 1], [200, 3], [199, 64], [33, 32]])
def test_prefixes_of_any_length(prefix):
    """Held to the sequence's length; a token sees the prefix's tokens that come behind it."""
    check(ref.Case(lens=[200, 64], news=[200, 7], heads=4, kv_heads=1, prefix=[min(max(p, 0), n) for p, n in zip(prefix, (200, 64))], seed=2))
    c = ref.Case(lens=[200, 64], news=[200, 7], heads=4, kv_heads=1, prefix=[min(max(p, 0), n) for p, n in zip(prefix, (200, 64))], seed=2)
    want, _, tol, _ = ref.attend(c)
    c.prefix = prefix
    out, _ = plan_of(c).forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c), prefix_lens=c.given()[1])
    compare(out, want, tol, "out")


@pytest.mark.parametrize("lens,news", [([5000], [1]), ([3001, 4100, 17], [1, 1, 1]), ([3500], [40]), ([2600], [300])])
def test_long(lens, news):
    check(ref.Case(lens=lens, news=news, heads=4, kv_heads=1, cap=10.0, slopes=[0.5, 0.1, 0.01, 0.0], page=128, seed=4))
    check(ref.Case(lens=lens, news=news, heads=4, kv_heads=1, first=docs_of(lens, news, 701), prefix=[100] * len(lens), page=128, seed=5))


@pytest.mark.parametrize("more", [dict(window=200, sinks=40, prefix=[130, 0, 900]), dict(prefix=[0, 700, 3]), dict(window=33, prefix=[1100, 0, 0]), dict(sinks=0, window=500), {}])
@pytest.mark.parametrize("docs", [0, 40, 333])
def test_keys_that_no_row_sees(more, docs):
    """Long contexts of which windows and documents leave little, of few rows and of many: what lies between the first keys and them is passed over."""
    lens, news = [2600, 1900, 1300], [300, 140, 5]
    first = docs_of(lens, news, docs) if docs else None
    check(ref.Case(lens=lens, news=news, heads=4, kv_heads=2, dim=64, first=first, cap=9.0, slopes=[0.2, 0.01, -0.001, 0.0] if docs != 40 else None, page=32, seed=docs, **more))
    first = [first[(7 * i) % len(first)] for i in range(len(first))] if docs else None    # in no order
    check(ref.Case(lens=lens, news=news, heads=4, kv_heads=2, dim=64, first=first, cap=9.0, page=32, seed=docs + 1, **more))


def test_packed_documents_are_sequences_of_their_own():
    """Documents one behind the other in one sequence and as sequences of a batch: the same, to the rounding of what is summed in which order."""
    sizes = [100, 33, 1, 257, 64, 130, 32, 7]
    L = sum(sizes)
    first = [sum(sizes[:i]) for i, n in enumerate(sizes) for _ in range(n)]
    out, lse = check(ref.Case(lens=[L], news=[L], heads=4, kv_heads=2, first=first, page=16, seed=6))
    c = ref.Case(lens=[L], news=[L], heads=4, kv_heads=2, page=16, seed=6)
    # the same rows as sequences: pages of one token's rows each are not possible, so the rows are appended to a pool of their own
    pages = [-(-n // 16) for n in sizes]
    table = torch.full((len(sizes), max(pages)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    pool = [torch.zeros(at, 2, 16, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    rows = [torch.stack([c.rows(x, 0, g)[0] for g in range(2)], dim=1).to(torch.bfloat16).cuda() for x in (c.k, c.v)]
    lens, starts = torch.tensor(sizes, dtype=torch.int32).cuda(), torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], dtype=torch.int32).cuda()
    plan = paged.PagedAttention(4, 128, kv_heads=2, dtype="bf16", page_size=16, max_batch=8, max_tokens=L)
    plan.append(*rows, *pool, table.cuda(), lens, starts)
    other, other_lse = plan.forward(c.q.cuda(), *pool, table.cuda(), lens, starts)
    _, _, tol, tol_lse = ref.attend(ref.Case(lens=[L], news=[L], heads=4, kv_heads=2, first=first, page=16, seed=6))
    compare(out, other.double().cpu(), 2 * tol, "out")
    compare(lse, other_lse.double().cpu(), 2 * tol_lse, "lse")


def test_hidden_places_may_hold_anything():
    """Infinities and NaN in K and V of keys that masks hide, in pages behind the end, and pages that are not there."""
    for lens, news in (([300], [300]), ([90, 64], [3, 1])):
        first = docs_of(lens, news, 50)
        c = ref.Case(lens=lens, news=news, heads=4, kv_heads=2, first=first, cap=4.0, seed=8)
        for x, bad in ((c.k, float("nan")), (c.v, float("inf")), (c.v, float("nan"))):
            # the last token of the last new one's document in front: hidden from the last document's tokens, seen by those in front
            j = max(0, first[-1] - 1)
            x[c.row(len(lens) - 1, j), :, j % c.page] = bad
        if news[0] > 1 and len(lens) == 1:
            c.table[0, 3] = -1
        plan = plan_of(c)
        out, lse = plan.forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c), first_keys=c.given()[2])
        want, want_lse, tol, tol_lse = ref.attend(c)
        T = sum(news)
        # rows that do not see that key are what they are; those that do are NaN
        j, b = max(0, first[-1] - 1), len(lens) - 1
        for t in range(T):
            of = 0 if t < news[0] else 1
            p = lens[of] - news[of] + (t - (0 if of == 0 else news[0]))
            if of == b and first[t] <= j <= p:
                assert out[t].isnan().all()
            else:
                compare(out[t], want[t], tol[t], t)
                compare(lse[:, t], want_lse[:, t], tol_lse[:, t], t)


@pytest.mark.parametrize("scores", ["documents", "cap and slopes", "window and prefix"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_long_chunks_walk_again_where_a_hidden_v_is_odd(scores, value):
    """Many rows: a V that is no number, in places that some rows of a workgroup see and others do not, and in places that none sees."""
    lens, news = [700], [420]
    more = SCORES[scores](dict(lens=lens, news=news, heads=4))
    c = ref.Case(lens=lens, news=news, heads=4, kv_heads=2, page=32, seed=12, **more)
    places = [5, 300, 431, 699]
    for j in places:
        c.v[c.row(0, j), :, j % 32, 7] = value
    c.k[c.row(0, 40), :, 40 % 32] = value if scores == "documents" else 0.5
    c.table[0, 4] = -1 if scores == "documents" else c.table[0, 4]
    plan = plan_of(c)
    slopes, prefix, first = c.given()
    out, lse = plan.forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c), prefix_lens=prefix, first_keys=first)
    want, want_lse, tol, tol_lse = ref.attend(c)
    compare(lse, want_lse, tol_lse, "lse")
    # (place 5 is seen by all rows but those of later documents: as one of the keys before, or of the prefix)
    assert torch.isfinite(want[:, :, 8:]).all() and not torch.isfinite(want[:, :, 7]).all() and (scores != "documents" or torch.isfinite(want[:, :, 7]).any())
    # A weight below 2^-126 is 0 in 32 bits, and 0 times an infinity is no number, where the definition has an infinity: under slopes that of a far key.
    faint = torch.zeros(420, 4, dtype=torch.bool)
    for h in range(4):
        k, there = c.rows(c.k, 0, h // 2)
        ok, x, _ = c.scores(0, h, k, there)
        faint[:, h] = (ok & (x - want_lse[h][:, None] < -125 * math.log(2)))[:, places].any(dim=1)
    assert scores != "documents" or not faint.any()
    assert not torch.isfinite(out[:, :, 7].cpu()[faint]).any()
    got = out.double().cpu()
    got[:, :, 7] = torch.where(faint, want[:, :, 7], got[:, :, 7])
    compare(got, want, tol, "out")


def test_a_cap_holds_infinite_scores():
    """Products past the range of 32 bits: the cap, of either sign."""
    c = ref.Case(lens=[64], news=[2], heads=2, kv_heads=2, cap=30.0, dtype="bf16", seed=3)
    c.q[:] = c.q.sign() * 1e25
    c.k[:] = torch.where(c.k.isnan(), c.k, torch.tensor(1e25, dtype=torch.bfloat16) * c.q[0, 0].sign() * (1 - 2 * (torch.arange(c.page) % 2)[None, None, :, None]))
    out, lse = plan_of(c).forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c))
    v, _ = c.rows(c.v, 0, 0)
    n = 63    # the first token sees 63 keys: the even ones score the cap, the odd ones its negative, which weighs e^-60
    want = v[:n:2].mean(dim=0)
    size = v[:n:2].abs().mean(dim=0)
    # equal weights, exactly; a sum of 32 and the rounding of O (the odd ones weigh 2^-86)
    assert ((out[0, 0].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * 2.0 ** -24 * size).all()
    assert abs(float(lse[0, 0]) - 30 - math.log(32)) < 2.0 ** -18


def test_no_scoring_is_the_plain_call():
    """Members that are 0 or NULL: the plain kernels' bits, through the C entry; masks that hide nothing: the same to the rounding."""
    import ctypes
    from ringattention_amd._lib import RingattnPagedScoring
    c = ref.Case(lens=[400, 33], news=[300, 1], heads=4, kv_heads=2, seed=5)
    plan = plan_of(c)
    q, k, v, seqs = c.q.cuda(), c.k.cuda(), c.v.cuda(), sequences(c)
    out, lse = plan.forward(q, k, v, *seqs)
    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
    cache = plan._cache(k, v, *seqs)
    for scoring in (None, RingattnPagedScoring(0.0, None, None, None)):
        rc = plan.lib.ringattn_paged_fwd_scored(plan.handle, ctypes.byref(cache), ctypes.byref(scoring) if scoring else None, q.data_ptr(), c.tokens,
                                                *paged._strides(q), o2.data_ptr(), *paged._strides(o2), l2.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(o2, out) and torch.equal(l2, lse)
        o2.zero_()
    zeros = torch.zeros(c.tokens, dtype=torch.int32, device="cuda")
    o3, l3 = plan.forward(q, k, v, *seqs, first_keys=zeros, prefix_lens=zeros[:2])
    _, _, tol, tol_lse = ref.attend(c)
    compare(o3, out.double().cpu(), 2 * tol, "out")
    compare(l3, lse.double().cpu(), 2 * tol_lse, "lse")


def test_parts_of_a_sequence_with_a_cap():
    """A sequence spread over two pools: capped partials without causality, put together by merge."""
    c = ref.Case(lens=[200], news=[1], heads=4, kv_heads=2, cap=6.0, seed=7)
    want, want_lse, tol, tol_lse = ref.attend(c)
    parts = []
    for first, last in ((0, 6), (6, 13)):
        plan = paged.PagedAttention(4, 128, kv_heads=2, dtype="bf16", page_size=16, max_batch=1, max_tokens=1, causal=False, partials=True, softcap=6.0)
        n = min(200, last * 16) - first * 16
        parts.append(plan.forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), c.table[:, first:last].cuda().contiguous(), torch.tensor([n], dtype=torch.int32).cuda(), c.starts.cuda()))
    o, lse = api.merge(torch.stack([p[0].reshape(4, 128) for p in parts]), torch.stack([p[1].reshape(4) for p in parts]), "bf16")
    compare(o.reshape(1, 4, 128), want, 2 * tol, "out")
    compare(lse.reshape(4, 1), want_lse, 2 * tol_lse + 2.0 ** -20, "lse")


def test_captured():
    """Lengths, prefixes and first keys are read at every replay."""
    c = ref.Case(lens=[300, 40, 90], news=[130, 1, 5], heads=4, kv_heads=2, cap=8.0, slopes=slopes_of(4), prefix=[10, 0, 90], first=docs_of([300, 40, 90], [130, 1, 5], 64), seed=1)
    plan = plan_of(c)
    slopes, prefix, first = c.given()
    q, k, v, (table, lens, starts) = c.q.cuda(), c.k.cuda(), c.v.cuda(), sequences(c)
    out, lse, scores = torch.empty_like(q), torch.empty(4, c.tokens, device="cuda"), torch.zeros(c.pages, 2, c.page, device="cuda")
    plan.forward(q, k, v, table, lens, starts, out, lse, prefix_lens=prefix, first_keys=first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.forward(q, k, v, table, lens, starts, out, lse, prefix_lens=prefix, first_keys=first)
        plan.weights(q, lse, k, table, lens, starts, scores, prefix_lens=prefix, first_keys=first)
    for shift in (0, 3, 17, 0):
        c.lens = [300 - shift, 40, 90 - shift]
        c.prefix = [10 + shift, shift, 90 - 2 * shift]
        c.first = [max(0, x - 5 * shift) for x in docs_of(c.lens, c.news, 64)]
        lens.copy_(c.kv_lens())
        prefix.copy_(torch.tensor(c.prefix, dtype=torch.int32))
        first.copy_(torch.tensor(c.first, dtype=torch.int32))
        scores.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse, tol, tol_lse = ref.attend(c)
        compare(out, want, tol, "out")
        compare(lse, want_lse, tol_lse, "lse")
        compare(scores, *ref.weights(c, lse.cpu()), "weights")


def test_streams_and_layouts():
    c = ref.Case(lens=[90, 64], news=[30, 2], heads=4, kv_heads=2, cap=5.0, prefix=[8, 64], seed=2)
    plan = plan_of(c)
    q = c.q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    wide = [torch.zeros(c.pages, c.page, 2, 136, dtype=torch.bfloat16, device="cuda") for _ in range(2)]   # token by token, rows with room between
    cache = [x.permute(0, 2, 1, 3)[..., :128] for x in wide]
    for x, given in zip(cache, (c.k, c.v)):
        x.copy_(given)
    prefix, args = c.given()[1], sequences(c)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    out, lse = plan.forward(q, *cache, *args, stream=stream, prefix_lens=prefix)
    stream.synchronize()
    want, want_lse, tol, tol_lse = ref.attend(c)
    compare(out, want, tol, "out")
    compare(lse, want_lse, tol_lse, "lse")


def test_pages_past_32_bits():
    """Pages behind the first 2^32 elements of a pool: the same bits as in a small one."""
    c = ref.Case(lens=[300, 40, 90], news=[130, 1, 5], heads=4, kv_heads=2, dim=64, cap=8.0, slopes=slopes_of(4), prefix=[10, 0, 90], first=docs_of([300, 40, 90], [130, 1, 5], 64), seed=4, spare=0.0)
    plan = plan_of(c)
    slopes, prefix, first = c.given()
    table, lens, starts = sequences(c)
    out, lse = plan.forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), table, lens, starts, prefix_lens=prefix, first_keys=first)
    scores = plan.weights(c.q.cuda(), lse, c.k.cuda(), table, lens, starts, torch.zeros(c.pages, 2, 16, device="cuda"), prefix_lens=prefix, first_keys=first)
    more = 2 ** 21 + 5    # pages of 2 x 16 x 64 in front
    k, v = (torch.cat((torch.zeros(more, *x.shape[1:], dtype=x.dtype, device="cuda"), x.cuda())) for x in (c.k, c.v))
    far = torch.where(table >= 0, table + more, table)
    out2, lse2 = plan.forward(c.q.cuda(), k, v, far, lens, starts, prefix_lens=prefix, first_keys=first)
    scores2 = plan.weights(c.q.cuda(), lse2, k, far, lens, starts, torch.zeros(more + c.pages, 2, 16, device="cuda"), prefix_lens=prefix, first_keys=first)
    assert torch.equal(out, out2) and torch.equal(lse, lse2) and torch.equal(scores, scores2[more:]) and not scores2[:more].any()


def test_refusals():
    c = ref.Case(lens=[40], news=[4], heads=4, kv_heads=2)
    q, k, v, seqs = c.q.cuda(), c.k.cuda(), c.v.cuda(), sequences(c)
    plan = plan_of(c)
    ints = torch.zeros(8, dtype=torch.int32, device="cuda")
    for bad in (dict(prefix_lens=ints), dict(prefix_lens=ints[:1].long()), dict(prefix_lens=ints[:1].cpu()), dict(first_keys=ints[:3]), dict(first_keys=ints[::2]),
                dict(first_keys=ints[:4].float())):
        with pytest.raises(ValueError):
            plan.forward(q, k, v, *seqs, **bad)
        with pytest.raises(ValueError):
            plan.weights(q, torch.zeros(4, 4, device="cuda"), k, *seqs, torch.zeros(c.pages, 2, 16, device="cuda"), **bad)
    open_plan = paged.PagedAttention(4, 128, kv_heads=2, dtype="bf16", page_size=16, causal=False)
    for bad in (dict(prefix_lens=ints[:1]), dict(first_keys=ints[:4])):
        with pytest.raises(ValueError, match="causal"):
            open_plan.forward(q, k, v, *seqs, **bad)
    for bad in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(softcap=2000.0), dict(slopes=torch.zeros(3, device="cuda")),
                dict(slopes=torch.zeros(4)), dict(slopes=torch.zeros(4, device="cuda"), causal=False)):
        with pytest.raises(ValueError):
            paged.PagedAttention(4, 128, kv_heads=2, dtype="bf16", page_size=16, **bad)
