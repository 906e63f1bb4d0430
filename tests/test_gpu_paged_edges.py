"""Calls of the paged cache's operators that their documentation allows and that are easily forgotten: sequences much shorter than the
call's tensors, rows that are not numbers, outputs over inputs, lengths and starts that are not true.  Against the definitions in 64 bits."""
import math

import pytest
import torch

import paged_reference as ref
from paged_reference import Case
from ringattention_amd import paged
from test_gpu_paged import check_forward, fill_scores, near, on_gpu, plan_for

pytestmark = pytest.mark.gpu

PADDED = 600   # rows of q of a call of one sequence, however few of them are its new tokens


def padded_case(dtype, dim, heads, hkv, new, room, window=0, sinks=0, seed=60, spare=float("nan")):
    """One sequence of 700 tokens, `new` of them new, q of PADDED rows; `room`: a table for 128 K tokens."""
    c = Case(dtype, dim, heads, hkv, 16, (700,), (new,), window=window, sinks=sinks, seed=seed, extra_rows=PADDED - new, spare=spare)
    if room:
        table = torch.full((1, 8192), -1, dtype=torch.int32)
        table[:, :c.table.shape[1]] = c.table
        c.table = table
    return c


def check_padded_forward(c, out, lse):
    new = c.news[0]
    o, z, tol, tol_z = ref.attend(c)
    near(out[:new], o[:new], tol[:new], "out")
    near(lse[:, :new], z[:, :new], tol_z[:, :new], "lse")
    assert (out[new:] == 7).all() and (lse[:, new:] == 7).all()


@pytest.mark.parametrize("new", [0, 1, 5, 31, 32, 33, 127, 128, 129, 300, 600])
@pytest.mark.parametrize("dtype,dim,heads,hkv,room,window,sinks", [("bf16", 128, 8, 2, False, 0, 0), ("fp16", 64, 4, 1, True, 0, 0), ("bf16", 64, 4, 4, True, 40, 3)])
def test_forward_of_one_sequence_of_fewer_tokens_than_rows(new, dtype, dim, heads, hkv, room, window, sinks):
    c = padded_case(dtype, dim, heads, hkv, new, room, window, sinks)
    out, lse = torch.full_like(c.q, 7.0).cuda(), torch.full((heads, PADDED), 7.0, device="cuda")
    plan_for(c).forward(c.q.cuda(), *on_gpu(c), out, lse)
    check_padded_forward(c, out, lse)


def test_captured_forward_of_a_prompts_last_chunk_and_next_tokens():
    """Captured for whole chunks of one prompt, replayed for its short last one, for single tokens, for nothing, and for a whole one again."""
    full = padded_case("bf16", 128, 8, 2, PADDED, True)
    plan, (k, v, table, lens, starts), q = plan_for(full), on_gpu(full), full.q.cuda()
    out, lse = torch.zeros_like(q), torch.zeros(8, PADDED, device="cuda")
    plan.forward(q, k, v, table, lens, starts, out, lse)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.forward(q, k, v, table, lens, starts, out, lse)
    for new in (20, 1, 0, 32, 33, PADDED, 1):
        c = padded_case("bf16", 128, 8, 2, new, True)
        q.copy_(c.q), k.copy_(c.k), v.copy_(c.v), table.copy_(c.table), starts.copy_(c.starts)
        out.fill_(7), lse.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_padded_forward(c, out, lse)
        again, lse_again = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
        plan.forward(q, k, v, table, lens, starts, again, lse_again)
        assert torch.equal(again, out) and torch.equal(lse_again, lse)


@pytest.mark.parametrize("new", [0, 1, 5, 47, 48, 49, 191, 192, 193, 600])
@pytest.mark.parametrize("dtype,dim,heads,hkv,room,window,sinks", [("bf16", 128, 8, 2, False, 0, 0), ("fp16", 64, 4, 1, True, 0, 0), ("bf16", 64, 4, 4, True, 40, 3)])
def test_weights_of_one_sequence_of_fewer_tokens_than_rows(new, dtype, dim, heads, hkv, room, window, sinks):
    c = padded_case(dtype, dim, heads, hkv, new, room, window, sinks, spare=0.0)
    lse = torch.zeros(heads, PADDED)
    lse[:, :new] = ref.attend(c)[1][:, :new]
    k, _, table, lens, starts = on_gpu(c)
    scores = torch.full((c.pages, hkv, 16), 0.5, device="cuda")
    plan_for(c).weights(c.q.cuda(), lse.cuda(), k, table, lens, starts, scores)
    w, off = ref.weights(c, lse)
    near(scores, w + 0.5, off + 2.0 ** -24 * (w + 0.5), "scores")


def test_captured_weights_of_a_prompts_last_chunk_and_next_tokens():
    full = padded_case("bf16", 128, 8, 2, PADDED, True, spare=0.0)
    plan, (k, _, table, lens, starts), q = plan_for(full), on_gpu(full), full.q.cuda()
    lse, scores = torch.zeros(8, PADDED, device="cuda"), torch.zeros(full.pages, 2, 16, device="cuda")
    plan.weights(q, lse, k, table, lens, starts, scores)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.weights(q, lse, k, table, lens, starts, scores)
    for new in (20, 1, 0, 48, 49, PADDED, 1):
        c = padded_case("bf16", 128, 8, 2, new, True, spare=0.0)
        z = torch.zeros(8, PADDED)
        z[:, :new] = ref.attend(c)[1][:, :new]
        starts.copy_(c.starts), lse.copy_(z), scores.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        w, off = ref.weights(c, z)
        near(scores, w, off, "scores")
        again = torch.zeros_like(scores)
        plan.weights(q, lse, k, table, lens, starts, again)
        assert torch.equal(again, scores)


@pytest.mark.parametrize("dim,lens,news", [(128, (1024, 1000), (460, 460)), (64, (1024, 1000), (512, 530))])
def test_shares_of_row_tiles_of_which_some_have_few_rows(dim, lens, news):
    """More pieces of row tiles to put together than workgroups do it, so that one has several in turn -- one with rows, one without, one with rows."""
    c = Case("bf16", dim, 32, 8, 64, lens, news, seed=66)
    plan, out, lse = check_forward(c)
    q, gpu = c.q.cuda(), on_gpu(c)
    for _ in range(20):
        again, lse_again = plan.forward(q, *gpu)
        assert torch.equal(again, out) and torch.equal(lse_again, lse)


@pytest.mark.parametrize("lens,budget,hkv", [((300, 20, 700, 64), 64, 4), ((21000, 9), 5000, 3), ((40,) * 200, 30, 8)])
def test_kept_lengths_in_place_of_the_lengths(lens, budget, hkv):
    """kept_lens may be kv_lens itself: a loop that goes on with the kept tokens has its lengths at once."""
    page = 16
    B, need = len(lens), [-(-n // page) for n in lens]
    pages = sum(need) + B * -(-budget // page)
    g = torch.Generator().manual_seed(64)
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(sum(need[:b]), sum(need[:b]) + n)
    kept_table = (torch.arange(pages - sum(need), dtype=torch.int32) + sum(need)).reshape(B, -1).cuda()
    k = torch.randn(pages, hkv, page, 64, generator=g).half().cuda()
    scores = torch.rand(pages, hkv, page, generator=g).cuda()
    results = []
    for same in (False, True):
        plan = plan_for(Case("fp16", 64, hkv, hkv, page, lens, (0,) * B, seed=65))
        kv_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        k2, v2, s2 = k.clone(), -k, scores.clone()
        kept = torch.full((B, hkv, budget), -7, dtype=torch.int32, device="cuda")
        kept_lens = kv_lens if same else torch.zeros_like(kv_lens)
        plan.evict(k2, v2, s2, table.cuda(), kv_lens, kept_table, budget, 2, 5, kept, kept_lens)
        results.append([x.cpu() for x in (k2, v2, s2, kept, kept_lens)])
    assert results[0][4].tolist() == [min(n, budget) for n in lens]
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_append_and_forward_take_the_same_places():
    """Lengths beyond the table and starts beyond the tokens are held to them, the same way by every call: what append wrote is what forward of the same
    call takes for the new tokens."""
    heads = hkv = 2
    B, cap, page, d, T = 4, 4, 16, 64, 30
    g = torch.Generator().manual_seed(62)
    for lens, starts in (([100, 64, 10 ** 9, 40], [0, 5, 9, 20, 30]), ([64, 30, 50, 60], [0, 5, 9, 20, 1000]), ([64, 30, 50, 2 ** 31 - 1], [-9, 5, 9, 20, 2 ** 31 - 1]),
                         ([30, 30, 30, 30], [0, 0, 0, 0, 31]), ([0, -5, 3, 64], [0, 2, 4, 9, 30])):
        c = Case("bf16", d, heads, hkv, page, (cap * page,) * B, (0,) * B, seed=63, spare=0.0, extra_rows=T)
        c.table = c.table[:, :cap].contiguous()
        c.q = torch.randn(T, heads, d, generator=g).bfloat16()
        new_k, new_v = (torch.randn(T, hkv, d, generator=g).bfloat16() for _ in range(2))
        k, v, table, _, _ = on_gpu(c)
        scores = torch.ones(c.pages, hkv, page, device="cuda")
        l, s = torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda()
        plan = plan_for(c)
        plan.append(new_k.cuda(), new_v.cuda(), k, v, table, l, s, scores)
        out, lse = torch.zeros(T, heads, d).bfloat16().cuda(), torch.zeros(heads, T, device="cuda")
        plan.forward(c.q.cuda(), k, v, table, l, s, out, lse)
        # the same with what is held to, by the definition
        c.lens = [min(max(n, 0), cap * page) for n in lens]
        held = [min(max(x, 0), T) for x in starts]
        c.starts, c.news = torch.tensor(held, dtype=torch.int32), [held[b + 1] - held[b] for b in range(B)]
        want_scores = torch.ones(c.pages, hkv, page)
        for b in range(B):
            for i in range(c.news[b]):
                j = c.lens[b] - c.news[b] + i
                if j >= 0:
                    p = c.row(b, j)
                    c.k[p, :, j % page], c.v[p, :, j % page], want_scores[p, :, j % page] = new_k[held[b] + i], new_v[held[b] + i], 0
        assert torch.equal(k.cpu(), c.k) and torch.equal(v.cpu(), c.v) and torch.equal(scores.cpu(), want_scores), (lens, starts)
        o, z, tol, tol_z = ref.attend(c)
        rows = torch.zeros(T, dtype=torch.bool)
        rows[held[0]:held[-1]] = True
        near(out[rows], o[rows], tol[rows], "out")
        near(lse[:, rows], z[:, rows], tol_z[:, rows], "lse")


def guarded(shape, dtype, value, room=1 << 18):
    """(a tensor filled with `value`, the memory it is a part of, where it lies): `room` elements of a value of their own on both sides."""
    n = math.prod(shape)
    whole = torch.full((n + 2 * room,), 77, dtype=dtype, device="cuda")
    whole[room:room + n] = value
    return whole[room:room + n].view(shape), whole, slice(room, room + n)


def untouched_outside(whole, inside):
    return bool((whole[:inside.start] == 77).all()) and bool((whole[inside.stop:] == 77).all())


def test_starts_that_go_up_and_down_thousands_of_times():
    """2048 sequences that all claim the call's 64 tokens, each over a million cached ones whose pages are not there: 5 x 2^30 key tiles in all, far
    more than tokens that are nobody's twice can have."""
    B, T, heads, page, cap = 4096, 64, 40, 1024, 1024
    plan = paged.PagedAttention(heads, 64, dtype="fp16", page_size=page, max_batch=B, max_tokens=T)
    table = torch.full((B, cap), -1, dtype=torch.int32, device="cuda")
    lens = torch.full((B,), cap * page, dtype=torch.int32, device="cuda")
    starts = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    starts[1::2] = T
    q = torch.zeros(T, heads, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(1, heads, page, 64, dtype=torch.float16, device="cuda")
    out, out_all, out_at = guarded((T, heads, 64), torch.float16, 5)
    lse, lse_all, lse_at = guarded((heads, T), torch.float32, 5)
    plan.forward(q, k, k, table, lens, starts, out, lse)
    torch.cuda.synchronize()
    assert untouched_outside(out_all, out_at) and untouched_outside(lse_all, lse_at)
    # and the plan's next call is as good as any
    starts.fill_(T)
    starts[0] = 0
    plan.forward(q, k, k, table, lens, starts, out, lse)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert untouched_outside(out_all, out_at) and untouched_outside(lse_all, lse_at)


@pytest.mark.parametrize("causal,window,sinks", [(True, 0, 0), (True, 40, 3), (True, 5, 0), (False, 0, 0)])
@pytest.mark.parametrize("lens,news", [((100, 40), (5, 30)), ((700,), (300,)), ((900, 90), (400, 1)), ((90, 33, 300), (1, 1, 1))])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_weights_of_rows_whose_lse_is_no_number(lens, news, causal, window, sinks, value):
    """Their weights are no numbers where they see a key (0 for -inf), and nothing where they do not: later tokens, tokens in front of the window."""
    for dtype, dim, heads, hkv in (("bf16", 128, 4, 2), ("fp16", 64, 3, 3)):
        c = Case(dtype, dim, heads, hkv, 16, lens, news, window=window, sinks=sinks, causal=causal, seed=61, spare=0.0)
        lse = ref.attend(c)[1].float()
        at = [int(c.starts[b]) + n // 2 for b, n in enumerate(news)]   # a token in the middle of each chunk, one head of it
        for i, t in enumerate(at):
            lse[i % heads, t] = value
        k, _, table, lens_, starts = on_gpu(c)
        scores = torch.zeros(c.pages, hkv, 16, device="cuda")
        plan_for(c).weights(c.q.cuda(), lse.cuda(), k, table, lens_, starts, scores)
        clean = lse.clone()
        for i, t in enumerate(at):
            clean[i % heads, t] = -math.inf
        w, off = ref.weights(c, clean)   # of all other rows
        if value == math.inf:            # exp(s - inf) = 0
            near(scores, w, off, "scores")
            continue
        for i, t in enumerate(at) if value != value else ():
            b, g = i, i % heads // (heads // hkv)
            _, there = c.rows(c.k, b, g)
            for j in c.seen(b, there)[t - int(c.starts[b])].nonzero().flatten().tolist():
                w[c.row(b, j), g, j % 16] = math.nan
        near(scores, w, off, "scores")


def kept_present(scores, there, budget, first, last):
    """Places that stay of one sequence's KV head where only tokens that are there do."""
    L, there = len(scores), there.tolist()
    if L <= budget:
        return [j for j in range(L) if there[j]]
    value = [-math.inf if math.isnan(x) else x for x in scores.tolist()]
    middle = sorted((j for j in range(first, L - last) if there[j]), key=lambda j: (-value[j], j))[:budget - first - last]
    return sorted([j for j in [*range(first), *range(L - last, L)] if there[j]] + middle)


@pytest.mark.parametrize("kind", ["exp", "odd", "zeros"])
@pytest.mark.parametrize("lens,budget,first,last,hkv", [((300, 20, 700, 64, 0), 64, 20, 33, 3), ((90, 17, 33), 40, 0, 0, 2), ((21000, 9, 9000), 5000, 4, 100, 2),
                                                        ((2100,) * 40, 1500, 100, 100, 1)])
def test_evict_keeps_only_tokens_that_are_there(kind, lens, budget, first, last, hkv):
    """Every third page is not there: no token of it stays, the lengths say so, and what goes on with the kept ones sees no row that nobody wrote."""
    page, d, B = 16, 64, len(lens)
    c = Case("bf16", d, hkv, hkv, page, lens, (0,) * B, seed=67, spare=0.0)
    c.table[:, ::3] = -1
    if B > 2:
        c.table[2, 5], c.table[1] = c.pages + 10 ** 6, -1     # of the second none is there at all
    scores = fill_scores(c, kind, 68)
    kept_pages = -(-budget // page)
    pages = c.pages + B * kept_pages
    kept_table = (torch.arange(B * kept_pages, dtype=torch.int32) + c.pages).reshape(B, -1)
    k, v = (torch.cat([x, torch.full((pages - c.pages, hkv, page, d), math.nan).to(x.dtype)]) for x in (c.k, c.v))
    s = torch.cat([scores, torch.full((pages - c.pages, hkv, page), 9.0)])
    plan = plan_for(c, keep_present=True)
    results = []
    for same in (False, True):
        gk, gv, gs, lens_ = k.cuda(), v.cuda(), s.cuda(), c.kv_lens().cuda()
        kept = torch.full((B, hkv, budget), 10 ** 9, dtype=torch.int32, device="cuda")
        kept_lens = lens_ if same else torch.zeros_like(lens_)
        plan.evict(gk, gv, gs, c.table.cuda(), lens_, kept_table.cuda(), budget, first, last, kept, kept_lens)
        results.append([x.cpu() for x in (gk.view(torch.int16), gv.view(torch.int16), gs.view(torch.int32), kept, kept_lens)])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    kept, kept_lens = results[0][3], results[0][4].tolist()
    for b, n in enumerate(lens):
        at = c.table[b].long()[torch.arange(n) // page]
        there = (at >= 0) & (at < c.pages)
        for h in range(hkv):
            places = kept_present(scores[at.clamp(0, c.pages - 1), h, torch.arange(n) % page], there, budget, first, last)
            assert kept[b, h].tolist() == places + [-1] * (budget - len(places)) and kept_lens[b] == len(places), (b, h)
            i, j = torch.arange(len(places)), torch.tensor(places, dtype=torch.long)
            to, row = kept_table[b].long()[i // page], i % page
            for x in (k, v, s):
                x[to, h, row] = x[at[j], h, j % page]
    for x, y in zip((k.view(torch.int16), v.view(torch.int16), s.view(torch.int32)), results[0]):
        assert torch.equal(x, y)
    # a step over the kept tokens
    after = Case("bf16", d, hkv, hkv, page, kept_lens, tuple(min(n, 1) for n in kept_lens), seed=69)
    after.k, after.v, after.table, after.pages = k, v, kept_table, pages
    check_forward(after)


def test_captured_eviction_of_tokens_that_are_there():
    page, hkv, B, cap, budget = 16, 2, 3, 80, 200
    g = torch.Generator().manual_seed(70)
    pages = B * cap + B * -(-budget // page)
    base = [torch.randn(pages, hkv, page, 64, generator=g).half().cuda() for _ in range(2)] + [torch.rand(pages, hkv, page, generator=g).cuda()]
    kept_table = (torch.arange(pages - B * cap, dtype=torch.int32) + B * cap).reshape(B, -1).cuda()
    table, lens = torch.zeros(B, cap, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    plan = paged.PagedAttention(4, 64, kv_heads=hkv, page_size=page, max_batch=B, max_tokens=4, keep_present=True)
    state = [x.clone() for x in base] + [torch.zeros(B, hkv, budget, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")]

    def step():
        k, v, s, kept, kept_lens = state
        plan.evict(k, v, s, table, lens, kept_table, budget, 3, 20, kept, kept_lens)

    def fresh():
        for x, y in zip(state, base + [-2, -2]):
            x.copy_(y) if isinstance(y, torch.Tensor) else x.fill_(y)

    step()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i, L in enumerate(([1000, 30, 0], [7, 1280, 250], [640, 200, 201])):
        t = torch.randperm(B * cap, generator=g).reshape(B, cap).int()
        t[torch.rand(B, cap, generator=g) < 0.1 * (i + 1)] = -1
        table.copy_(t), lens.copy_(torch.tensor(L, dtype=torch.int32))
        fresh()
        step()
        torch.cuda.synchronize()
        eager = [x.clone() for x in state]
        fresh()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(state, eager)), L
        assert (state[4] <= torch.tensor(L, device="cuda")).all() and ((state[3] >= 0).sum(dim=2) == state[4][:, None]).all()


@pytest.mark.parametrize("lens,starts", [([10 ** 9, -5, 2 ** 31 - 1], [0, 3, 43, 45]), ([60, 90, 40], [0, 3, 400, 2 ** 31 - 1]), ([60, 90, 40], [-7, 30, 3, 45]),
                                         ([-2 ** 31, 90, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 45]), ([60, 90, 40], [45, 45, 45, 45]), ([1, 0, 2], [0, 20, 20, 45])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (17, 3)])
def test_lengths_that_are_not_true_write_nothing_else(lens, starts, window, sinks):
    """Lengths and starts of any kind: rows that no sequence has, places that no token has and what lies around the tensors stay as they were, and
    sequences whose lengths and starts, held to the table and the tokens, are ones of their own get what is theirs."""
    heads, hkv, page, d, T, budget = 4, 2, 16, 64, 45, 20
    c = Case("bf16", d, heads, hkv, page, (60, 90, 40), (3, 40, 2), window=window, sinks=sinks, seed=14, spare=0.0, extra_pages=8)
    held = [min(max(x, 0), T) for x in starts]
    c.starts = torch.tensor(held, dtype=torch.int32)
    c.news = [max(0, held[b + 1] - held[b]) for b in range(3)]
    room = c.table.shape[1] * page
    c.lens = [min(max(n, 0), room) for n in lens]
    plan = plan_for(c)
    assert c.tokens == T
    l, s = torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda()
    table, q = c.table.cuda(), c.q.cuda()
    of = [guarded(c.k.shape, torch.bfloat16, 0) for _ in range(2)] + [guarded((c.pages, hkv, page), torch.float32, 0.5)]
    (k, v, scores), places = [x[0] for x in of], [x[1:] for x in of]
    k.copy_(c.k), v.copy_(c.v)
    out, *out_at = guarded((T, heads, d), torch.bfloat16, 5)
    lse, *lse_at = guarded((heads, T), torch.float32, 5)
    plan.forward(q, k, v, table, l, s, out, lse)
    claims = torch.zeros(T, dtype=torch.int64)
    for b in range(3):
        claims[held[b]:held[b] + c.news[b]] += 1
    o, z, tol, tol_z = ref.attend(c)
    one = claims == 1
    near(out[one], o[one], tol[one], "out")
    near(lse[:, one], z[:, one], tol_z[:, one], "lse")
    assert (out[claims == 0] == 5).all() and (lse[:, claims == 0] == 5).all()
    # the weights, by an LSE of every row that is claimed once; rows of several sequences weigh nothing
    z = torch.where(one, z.float(), -math.inf)
    plan.weights(q, z.cuda(), k, table, l, s, scores)
    w, off = ref.weights(c, z)
    near(scores, w + 0.5, off + 2.0 ** -24 * (w + 0.5), "scores")
    # new rows: where append may write
    new = torch.full((T, hkv, d), 3.0, dtype=torch.bfloat16, device="cuda")
    plan.append(new, new, k, v, table, l, s, scores)
    want = c.k.clone()
    for b in range(3 if int(claims.max()) < 2 else 0):
        for j in range(max(0, c.lens[b] - c.news[b]), c.lens[b]):
            if c.row(b, j) is not None:
                want[c.row(b, j), :, j % page] = 3
    owned = torch.zeros(c.pages, page, dtype=torch.bool)   # any place that a sequence's table gives it
    for b in range(3):
        for j in range(c.lens[b]):
            if c.row(b, j) is not None:
                owned[c.row(b, j), j % page] = True
    if int(claims.max()) < 2:
        assert torch.equal(k.cpu(), want)
    assert torch.equal(k.cpu().transpose(1, 2)[~owned], c.k.transpose(1, 2)[~owned]) and torch.equal(v.cpu().transpose(1, 2)[~owned], c.v.transpose(1, 2)[~owned])
    free = [p for p in range(c.pages) if not (c.table == p).any()]
    kept_table = torch.tensor(free[:6], dtype=torch.int32).reshape(3, 2).cuda()
    kept, *kept_at = guarded((3, hkv, budget), torch.int32, -9)
    kept_lens, *lens_at = guarded((3,), torch.int32, -9)
    plan.evict(k, v, scores, table, l, kept_table, budget, 2, 5, kept, kept_lens)
    assert kept_lens.tolist() == [min(n, budget) for n in c.lens]
    assert ((kept >= 0).sum(dim=2).cpu() == torch.tensor(c.lens)[:, None].clamp(max=budget)).all()
    torch.cuda.synchronize()
    assert all(untouched_outside(*x) for x in places + [out_at, lse_at, kept_at, lens_at])


@pytest.mark.parametrize("dtype,dim,heads,sigma,seed", [("fp16", 128, 99, 3.0, 5113), ("fp16", 128, 99, 1.0, 72), ("bf16", 64, 24, 3.0, 73)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("lens,news,causal,lost", [((469, 235, 358, 455, 473), (120, 43, 90, 187, 79), False, True), ((900, 777), (300, 400), True, False)])
def test_the_same_bits_whatever_lies_behind_the_last_token(lens, news, causal, lost, value, dtype, dim, heads, sigma, seed):
    """An infinity or a NaN in a hidden place changes how masked tiles are multiplied, from its own tile on and from no other, in every run."""
    c = Case(dtype, dim, heads, 3, 256, lens, news, causal=causal, seed=seed, spare=value, sigma=sigma)
    if lost:
        c.table[2, 0] = -1
    plan, out, lse = check_forward(c)
    q, gpu = c.q.cuda(), on_gpu(c)
    for _ in range(20):
        again, lse_again = plan.forward(q, *gpu)
        assert torch.equal(again, out) and torch.equal(lse_again, lse)
