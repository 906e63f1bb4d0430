"""The paged cache's operators (ringattention_amd/paged.py) on the GPU against their definitions in 64 bits."""
import math

import pytest
import torch

import paged_reference as ref
from paged_reference import TORCH, Case
from ringattention_amd import api, paged

pytestmark = pytest.mark.gpu


def plan_for(c, **more):
    return paged.PagedAttention(c.heads, c.dim, kv_heads=c.kv_heads, dtype=c.dtype, page_size=c.page, max_batch=max(1, len(c.lens)),
                                max_tokens=max(1, c.tokens), causal=c.causal, window=c.window, sinks=c.sinks, **more)


def on_gpu(c):
    return c.k.cuda(), c.v.cuda(), c.table.cuda(), c.kv_lens().cuda(), c.starts.cuda()


def near(x, y, tol, what):
    x = x.double().cpu()
    assert x.shape == y.shape, what
    same = (x == y) | (x.isnan() & y.isnan())
    off = torch.where(same, 0.0, (x - y).abs())
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), off[bad].max().item(), (off / tol.clamp(min=1e-300))[bad].max().item(), bad.nonzero()[:4].tolist())


def check_forward(c, **more):
    plan = plan_for(c, **more)
    out, lse = plan.forward(c.q.cuda(), *on_gpu(c))
    torch.cuda.synchronize()
    o, z, tol, tol_z = ref.attend(c)
    rows = int(c.starts[-1])
    near(out[:rows], o[:rows], tol[:rows], "out")
    near(lse[:, :rows], z[:, :rows], tol_z[:, :rows], "lse")
    return plan, out, lse


RAGGED = [
    # lens, news: single tokens; chunks; sequences with nothing new, with nothing cached, with more new tokens than the cache has
    ((1,), (1,)), ((2, 1), (1, 1)), ((33, 64, 16, 31, 15), (1, 1, 1, 1, 1)), ((40, 0, 17, 3), (7, 0, 0, 3)),
    ((64, 5, 0), (64, 9, 4)), ((129, 300, 77), (2, 131, 77)), ((700,), (1,)), ((515, 260), (33, 260)), ((1000,), (650,)),
]


@pytest.mark.parametrize("lens,news", RAGGED)
@pytest.mark.parametrize("dtype,dim,heads,kv_heads,page", [("bf16", 128, 4, 2, 16), ("fp16", 64, 6, 6, 32), ("fp16", 128, 8, 1, 64), ("bf16", 64, 5, 1, 256)])
def test_forward(lens, news, dtype, dim, heads, kv_heads, page):
    check_forward(Case(dtype, dim, heads, kv_heads, page, lens, news, seed=len(lens)))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 4), (33, 40), (100, 0), (257, 65), (5000, 4)])
@pytest.mark.parametrize("lens,news", [((90, 1, 300), (1, 1, 1)), ((90, 33, 300), (50, 33, 7)), ((820,), (400,)), ((600, 900), (1, 530))])
def test_forward_with_a_window_and_sinks(window, sinks, lens, news):
    check_forward(Case("bf16", 128, 4, 2, 16, lens, news, window=window, sinks=sinks, seed=3))
    check_forward(Case("fp16", 64, 4, 1, 64, lens, news, window=window, sinks=sinks, seed=4))


@pytest.mark.parametrize("lens,news", RAGGED)
def test_forward_without_the_causal_mask(lens, news):
    check_forward(Case("bf16", 64, 8, 2, 32, lens, news, causal=False, seed=5))
    check_forward(Case("fp16", 128, 4, 4, 16, lens, news, causal=False, seed=6))


def test_many_sequences():
    lens = [(i * 37) % 150 for i in range(200)]
    news = [min(n, (i * 7) % 5) for i, n in enumerate(lens)]
    check_forward(Case("bf16", 64, 4, 2, 16, lens, news, seed=7))


@pytest.mark.parametrize("sigma", [0.05, 4.0, 12.0])
def test_forward_over_flat_and_peaked_scores(sigma):
    check_forward(Case("bf16", 128, 4, 2, 16, (300, 555), (1, 280), sigma=sigma, seed=8))
    check_forward(Case("fp16", 64, 4, 2, 16, (300, 555), (1, 280), sigma=sigma, seed=9))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_values_in_hidden_places_reach_nobody(value, window, sinks):
    """Behind a sequence's end, in pages of nobody, in front of the window, and in later tokens of the same chunk."""
    c = Case("bf16", 128, 4, 2, 16, (75, 300, 420), (1, 90, 300), window=window, sinks=sinks, seed=10, spare=value)
    for b, j in ((1, 250), (1, 298), (2, 200), (2, 333)):   # new tokens: earlier ones of the chunk do not see them
        p = c.row(b, j)
        c.v[p, :, j % 16, 5] = value
        c.v[p, 0, j % 16, 64:] = value
    check_forward(c)
    c = Case("fp16", 64, 2, 2, 32, (75, 300, 420), (1, 90, 300), window=window, sinks=sinks, seed=11, spare=value)
    for b, j in ((1, 250), (2, 419)):
        c.k[c.row(b, j), :, j % 32] = value
        c.v[c.row(b, j), :, j % 32] = value
    plan = plan_for(c)
    out, lse = plan.forward(c.q.cuda(), *on_gpu(c))
    o, z, tol, tol_z = ref.attend(c)
    # rows that see those keys: a score of plus or minus infinity or NaN, whichever the signs of q make it; the others as always
    sees = torch.zeros(c.tokens, dtype=torch.bool)
    for b, j in ((1, 250), (2, 419)):
        first = int(c.starts[b]) + j - (c.lens[b] - c.news[b])
        sees[first:int(c.starts[b + 1])] = True
    near(out[~sees.cuda()], o[~sees], tol[~sees], "out")
    near(lse[:, ~sees.cuda()], z[:, ~sees], tol_z[:, ~sees], "lse")


def test_pages_that_are_not_there():
    """-1, far negative, the first number past the pool, far past it: their tokens are hidden; behind a window nobody asks for them."""
    c = Case("bf16", 128, 4, 2, 16, (200, 333, 48), (1, 70, 48), seed=12)
    c.table[0, 3], c.table[0, 12], c.table[1, 0], c.table[1, 19] = -1, c.pages, -2 ** 31, 2 ** 31 - 1
    c.table[2, :3] = -7   # none at all: rows that see nothing
    _, out, lse = check_forward(c)
    assert (out[71:] == 0).all() and (lse[:, 71:] == -math.inf).all()
    # the same values whether the pages behind a window are there or not
    c = Case("fp16", 64, 4, 2, 32, (700, 650), (1, 200), window=64, sinks=5, seed=13)
    _, out, lse = check_forward(c)
    c.table[0, 1:19] = -1
    c.table[1, 1:11] = -1
    _, out2, lse2 = check_forward(c)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("lost", [2048, 2047, 2079, 4096, 31, 4000])
@pytest.mark.parametrize("new", [1, 140])
def test_a_page_that_is_not_there_far_into_a_sequence(lost, new):
    """Around the places where the pages of the next 64 key tiles are looked up."""
    c = Case("bf16", 64, 2, 1, 16, (4500,), (new,), seed=36)
    c.table[0, lost // 16] = -1
    check_forward(c)
    c = Case("fp16", 128, 2, 1, 16, (4500,), (new,), seed=37)
    c.table[0, lost // 16] = 2 ** 30
    plan, _, lse = check_forward(c)
    k, _, table, lens, starts = on_gpu(c)
    scores = torch.zeros(c.pages, 1, 16, device="cuda")
    plan.weights(c.q.cuda(), lse, k, table, lens, starts, scores)
    clean = Case("fp16", 128, 2, 1, 16, (4500,), (new,), seed=37, spare=0.0)
    clean.table[0, lost // 16] = -1
    w, off = ref.weights(clean, lse.cpu())
    near(scores, w, off, "scores")


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [4400, 4431, 4499])
def test_odd_values_in_a_long_chunk(value, at):
    """V of a new token that earlier ones of the chunk do not see, in every place of a tile's pair."""
    for dtype, dim in (("bf16", 128), ("fp16", 64)):
        c = Case(dtype, dim, 4, 2, 16, (4500,), (400,), seed=38)
        c.v[c.row(0, at), :, at % 16, 3] = value
        check_forward(c)


def test_lengths_that_are_not_true_stay_within_the_tensors():
    """Lengths beyond the table, negative ones, starts beyond the tokens or descending: nothing is read or written outside."""
    c = Case("bf16", 64, 4, 2, 16, (60, 90, 40), (3, 40, 2), seed=14)
    plan = plan_for(c)
    k, v, table, lens, starts = on_gpu(c)
    q = c.q.cuda()
    for bad_lens, bad_starts in (([10 ** 9, -5, 2 ** 31 - 1], [0, 3, 43, 45]), ([60, 90, 40], [0, 3, 400, 2 ** 31 - 1]), ([60, 90, 40], [-7, 30, 3, 45])):
        l, s = torch.tensor(bad_lens, dtype=torch.int32).cuda(), torch.tensor(bad_starts, dtype=torch.int32).cuda()
        out, lse = plan.forward(q, k, v, table, l, s)
        scores = torch.zeros(c.pages, 2, 16, device="cuda")
        plan.weights(q, lse.nan_to_num(0, 0, 0), k, table, l, s, scores)
        plan.append(q[:, :2], q[:, 2:], k.clone(), v.clone(), table, l, s, scores)
    torch.cuda.synchronize()


def test_rows_behind_the_last_sequence_are_left_alone():
    c = Case("bf16", 128, 4, 2, 16, (50, 200), (1, 64), seed=15, extra_rows=9)
    plan = plan_for(c)
    out, lse = torch.full_like(c.q, 7.0).cuda(), torch.full((4, c.tokens), 7.0, device="cuda")
    plan.forward(c.q.cuda(), *on_gpu(c), out, lse)
    assert (out[65:] == 7).all() and (lse[:, 65:] == 7).all()
    o, z, tol, tol_z = ref.attend(c)
    near(out[:65], o[:65], tol[:65], "out")


@pytest.mark.parametrize("news", [(1, 1), (3, 140)])
def test_strides(news):
    """Heads before tokens, q out of a tensor that holds q, k and v together, caches with tokens before heads, and K and V in one."""
    c = Case("bf16", 64, 4, 2, 16, (61, 333), news, seed=16)
    plan, out, lse = check_forward(c)
    k, v, table, lens, starts = on_gpu(c)
    q = c.q.cuda()
    T = c.tokens
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    fused = torch.cat([q, q + 1, q - 1], dim=1)[:, :4]
    by_token = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    both = torch.stack([k, v], dim=1)
    wide = torch.zeros(c.pages, 2, 16, 128, dtype=k.dtype, device="cuda")
    wide[..., :64], wide[..., 64:] = k, v
    for qq in (q, by_head, fused):
        for kk, vv in ((k, v), by_token, (both[:, 0], both[:, 1]), (wide[..., :64], wide[..., 64:])):
            o2, z2 = plan.forward(qq, kk, vv, table, lens, starts)
            assert torch.equal(o2, out) and torch.equal(z2, lse)
    to = torch.full((4, T + 3, 96), 5.0, dtype=q.dtype, device="cuda")   # heads first, rows further apart than they are long
    plan.forward(q, k, v, table, lens, starts, to[:, 1:T + 1, :64].transpose(0, 1), lse)
    assert torch.equal(to[:, 1:T + 1, :64].transpose(0, 1), out) and (to[:, 0] == 5).all() and (to[:, T + 1:] == 5).all() and (to[..., 64:] == 5).all()
    wide_table = torch.full((2, 40), -3, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    o2, _ = plan.forward(q, k, v, wide_table[:, :table.shape[1]], lens, starts)
    assert torch.equal(o2, out)


def test_a_pool_beyond_32_bits():
    """Pages that begin past 2^32 elements of the pool."""
    page, hkv, d = 64, 8, 128
    c = Case("bf16", d, 8, hkv, page, (1000, 150), (1, 150), seed=17, extra_pages=0)
    pages = 2 ** 32 // (page * hkv * d) + 300
    k = torch.empty(pages, hkv, page, d, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    far = torch.arange(c.pages, device="cuda") * 3 + pages - 3 * c.pages
    k[far], v[far] = c.k.cuda(), c.v.cuda()
    table = torch.where(c.table >= 0, far.cpu().int()[c.table.clamp(min=0).long()], -1).int().cuda()
    plan = plan_for(c)
    lens, starts = c.kv_lens().cuda(), c.starts.cuda()
    out, lse = plan.forward(c.q.cuda(), k, v, table, lens, starts)
    o, z, tol, tol_z = ref.attend(c)
    near(out, o, tol, "out")
    near(lse, z, tol_z, "lse")
    scores = torch.zeros(pages, hkv, page, device="cuda")
    plan.weights(c.q.cuda(), lse, k, table, lens, starts, scores)
    w, off = ref.weights(c, lse.cpu())
    near(scores[far], w, off, "scores")
    new = torch.randn(c.tokens, hkv, d, device="cuda").bfloat16()
    plan.append(new, -new, k, v, table, lens, starts, scores)
    for b, j, t in ((0, 999, 0), (1, 0, 1), (1, 149, 150)):
        p = int(table[b, j // page])
        assert torch.equal(k[p, :, j % page], new[t]) and torch.equal(v[p, :, j % page], -new[t]) and (scores[p, :, j % page] == 0).all()


def test_partials_of_two_pools_merge_into_the_whole():
    """A sequence whose first part lies in another pool: that one without the mask, its own part with it, merged by their LSEs."""
    c = Case("bf16", 128, 4, 2, 16, (700,), (300,), seed=18)
    whole, out, lse = check_forward(c)
    first = Case("bf16", 128, 4, 2, 16, (320,), (300,), causal=False, seed=18)
    first.k, first.v, first.pages, first.table, first.q = c.k, c.v, c.pages, c.table[:, :20].contiguous(), c.q
    rest = Case("bf16", 128, 4, 2, 16, (380,), (300,), seed=18)
    rest.k, rest.v, rest.pages, rest.table, rest.q = c.k, c.v, c.pages, c.table[:, 20:].contiguous(), c.q
    o, z = [], []
    for part in (first, rest):
        x, y = plan_for(part, partials=True).forward(part.q.cuda().transpose(0, 1).contiguous().transpose(0, 1), *on_gpu(part))
        assert x.dtype == torch.float32
        o.append(x.transpose(0, 1).reshape(-1, 128))
        z.append(y.reshape(-1))
    merged, merged_lse = api.merge(torch.stack(o).contiguous(), torch.stack(z), torch.bfloat16)
    o64, z64, tol, tol_z = ref.attend(c)
    near(merged.reshape(4, 300, 128).transpose(0, 1), o64, tol, "out")
    near(merged_lse.reshape(4, 300), z64, 2 * tol_z, "lse")


def test_a_prompt_as_the_ring_forward_has_it():
    """A whole prompt over the cache and the engine's forward over the same rows, both near the definition."""
    S = 640
    c = Case("fp16", 128, 4, 2, 64, (S,), (S,), seed=19)
    _, out, lse = check_forward(c)
    k = torch.stack([c.rows(c.k, 0, g)[0] for g in range(2)])[None].half().cuda()
    v = torch.stack([c.rows(c.v, 0, g)[0] for g in range(2)])[None].half().cuda()
    ring = api.RingAttention(2, [320, 320], 128, 1, 4, "fp16", True, kv_heads=2)
    o2, z2 = ring.forward(c.q.cuda().transpose(0, 1).contiguous()[None], k, v)
    _, _, tol, tol_z = ref.attend(c)
    near(o2[0].transpose(0, 1), out.double().cpu(), 2 * tol, "out")
    near(z2[0], lse.double().cpu(), 2 * tol_z, "lse")


@pytest.mark.parametrize("lens,news", RAGGED)
@pytest.mark.parametrize("window,sinks,causal", [(0, 0, True), (40, 3, True), (0, 0, False)])
def test_weights(lens, news, window, sinks, causal):
    for dtype, dim, heads, hkv, page in (("bf16", 128, 4, 2, 16), ("fp16", 64, 8, 1, 64)):
        c = Case(dtype, dim, heads, hkv, page, lens, news, window=window, sinks=sinks, causal=causal, seed=20)
        plan = plan_for(c)
        gpu = on_gpu(c)
        q = c.q.cuda()
        _, lse = plan.forward(q, *gpu)
        scores = torch.zeros(c.pages, hkv, page, device="cuda")
        plan.weights(q, lse, gpu[0], *gpu[2:], scores)
        clean = Case(dtype, dim, heads, hkv, page, lens, news, window=window, sinks=sinks, causal=causal, seed=20, spare=0.0)
        w, off = ref.weights(clean, lse.cpu())
        near(scores, w, off, "scores")
        again = torch.ones_like(scores)   # added to what is there, the same in every run
        plan.weights(q, lse, gpu[0], *gpu[2:], again)
        assert torch.equal(again, 1 + scores)


@pytest.mark.parametrize("dtype,dim,heads,hkv,page", [("bf16", 128, 8, 2, 16), ("fp16", 64, 3, 3, 64)])
@pytest.mark.parametrize("lens,news,window,sinks,causal", [((1100,), (1100,), 0, 0, True), ((1100, 90, 700), (300, 1, 700), 0, 0, True), ((900, 513), (800, 513), 130, 70, True),
                                                           ((1500, 40), (257, 200), 0, 0, False), ((333, 1290), (333, 129), 1, 0, True)])
def test_weights_of_long_chunks(dtype, dim, heads, hkv, page, lens, news, window, sinks, causal):
    c = Case(dtype, dim, heads, hkv, page, lens, news, window=window, sinks=sinks, causal=causal, seed=33)
    c.table[0, 2] = -1
    plan = plan_for(c)
    gpu = on_gpu(c)
    _, lse = plan.forward(c.q.cuda(), *gpu)
    scores = torch.zeros(c.pages, hkv, page, device="cuda")
    plan.weights(c.q.cuda(), lse, gpu[0], *gpu[2:], scores)
    clean = Case(dtype, dim, heads, hkv, page, lens, news, window=window, sinks=sinks, causal=causal, seed=33, spare=0.0)
    clean.table[0, 2] = -1
    w, off = ref.weights(clean, lse.cpu())
    near(scores, w, off, "scores")


@pytest.mark.parametrize("dtype,dim,heads,lens", [("bf16", 128, 8, (8600, 9000, 300)), ("fp16", 64, 4, (8704,)), ("bf16", 64, 32, (16900, 40))])
def test_parts_by_the_dozen(dtype, dim, heads, lens):
    # one KV head: the keys of a row go to more workgroups than one puts together, the last of which is alone or begins the next sequence's
    c = Case(dtype, dim, heads, 1, 64, lens, (1,) * len(lens), seed=42)
    check_forward(c)
    plan = plan_for(c)
    gpu = on_gpu(c)
    out, lse = plan.forward(c.q.cuda(), *gpu)
    for _ in range(3):
        again, lse_again = plan.forward(c.q.cuda(), *gpu)
        assert torch.equal(out, again) and torch.equal(lse, lse_again)


@pytest.mark.parametrize("dtype,dim,heads,lens,news", [("bf16", 128, 16, (20000,), (16,)), ("fp16", 64, 8, (9000, 5000), (40, 17))])
def test_shares_by_the_dozen(dtype, dim, heads, lens, news):
    c = Case(dtype, dim, heads, 1, 64, lens, news, seed=43)   # many rows, and their keys in dozens of shares
    check_forward(c)
    plan = plan_for(c)
    gpu = on_gpu(c)
    out, lse = plan.forward(c.q.cuda(), *gpu)
    again, lse_again = plan.forward(c.q.cuda(), *gpu)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)


@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 0), (40, 3)])
@pytest.mark.parametrize("dtype,dim,heads,hkv,batch,longest", [("bf16", 128, 16, 8, 60, 130), ("fp16", 64, 12, 12, 150, 40), ("bf16", 64, 32, 16, 50, 500)])
def test_small_sequences_by_the_hundred(dtype, dim, heads, hkv, batch, longest, window, sinks):
    # more row tiles than workgroups: those that see little are a wave's own, eight in a row or fewer, those that see more are not; sequences
    # without anything new or without anything cached in between, pages that are not there, odd values in hidden places
    lens = [(7 * i * i + 3 * i) % longest if i % 9 else longest * (i % 18 == 0) for i in range(batch)]
    news = [0 if i % 11 == 3 else 1 + (i % 5 == 0) * (i % 7) for i in range(batch)]
    for odd in (0.0, math.nan):
        c = Case(dtype, dim, heads, hkv, 16, lens, news, window=window, sinks=sinks, seed=44, spare=odd)
        if c.table.shape[1] > 2:
            c.table[batch // 2, 1] = -1
        _, out, lse = check_forward(c)
        plan = plan_for(c)
        again, lse_again = plan.forward(c.q.cuda(), *on_gpu(c))
        rows = int(c.starts[-1])
        assert torch.equal(out[:rows], again[:rows]) and torch.equal(lse[:, :rows], lse_again[:, :rows])


@pytest.mark.parametrize("lens,news", [((5000, 70, 0, 2100), (1, 1, 0, 1)), ((40,) * 12, (1,) * 12), ((3000, 9, 1500), (40, 9, 130))])
def test_tables_with_room_for_very_long_sequences(lens, news):
    # 2^30 tokens a sequence: the key tiles that there might be are dealt out several at a time, the few that there are all the same
    c = Case("fp16", 64, 32, 32, 1024, lens, news, seed=45)
    wide = torch.full((len(lens), 1 << 20), -1, dtype=torch.int32)
    wide[:, :c.table.shape[1]] = c.table
    plan = plan_for(c)
    k, v, table, kv_lens, starts = on_gpu(c)
    out, lse = plan.forward(c.q.cuda(), k, v, wide.cuda(), kv_lens, starts)
    o, z, tol, tol_z = ref.attend(c)
    rows = int(c.starts[-1])
    near(out[:rows], o[:rows], tol[:rows], "out")
    near(lse[:, :rows], z[:, :rows], tol_z[:, :rows], "lse")


@pytest.mark.parametrize("dtype,dim,heads,hkv,lens,new,window", [("fp16", 64, 8, 1, (2000,) * 80, 1, 0), ("bf16", 128, 16, 8, (10000,), 24, 0), ("bf16", 64, 8, 8, (6000,) * 2, 3, 0),
                                                                   ("fp16", 128, 32, 4, (5003,) * 5, 1, 0), ("fp16", 64, 16, 16, (4096,), 33, 2100)])
def test_sequences_as_long_as_each_other(dtype, dim, heads, hkv, lens, new, window):
    # their row tiles are cut into as many runs each, with a row tile counting as more than it sees where that does not go up
    c = Case(dtype, dim, heads, hkv, 64, lens, (new,) * len(lens), window=window, seed=53)
    c.table[0, 3] = -1
    check_forward(c)
    plan, gpu = plan_for(c), on_gpu(c)
    out, lse = plan.forward(c.q.cuda(), *gpu)
    again, lse_again = plan.forward(c.q.cuda(), *gpu)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)
    # one of them shorter than the others
    c.lens[-1] -= 1500
    check_forward(c)


def with_room(c, tokens=1 << 21):
    """The same sequences in tables that might hold much longer ones: which kernel has what goes by what a call may hold."""
    more = torch.full((len(c.lens), tokens // c.page - c.table.shape[1]), -1, dtype=torch.int32)
    c.table = torch.cat([c.table, more], 1)
    return c


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 0), (130, 35)])
@pytest.mark.parametrize("lens,news", RAGGED + [((333, 90), (130, 66)), ((2200,), (70,)), ((515, 2, 700), (300, 1, 64))])
def test_forward_in_tables_with_room(lens, news, window, sinks):
    for dtype, dim, heads, hkv, page in (("bf16", 128, 8, 2, 16), ("fp16", 64, 4, 1, 64)):
        check_forward(with_room(Case(dtype, dim, heads, hkv, page, lens, news, window=window, sinks=sinks, seed=50)))


@pytest.mark.parametrize("lost", [2048, 2047, 31, 4000])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_missing_pages_and_odd_values_in_tables_with_room(lost, value):
    c = with_room(Case("bf16", 128, 4, 2, 16, (4200,), (140,), seed=51))
    c.table[0, lost // 16] = -1
    c.v[int(c.table[0, 4195 // 16]), :, 4195 % 16:] = value   # hidden from all but the last rows
    check_forward(c)
    c = with_room(Case("fp16", 64, 8, 2, 32, (900, 300), (100, 90), window=100, sinks=3, seed=52))
    c.v[int(c.table[0, 20]), :, 5:] = value                   # behind the windows of most rows
    check_forward(c)


@pytest.mark.parametrize("dtype,dim,heads,hkv,lens,news,causal", [("bf16", 128, 8, 2, (2000,), (2000,), True), ("fp16", 64, 8, 1, (2100, 700), (2000, 600), False),
                                                                  ("fp16", 64, 256, 32, (128,) * 10, (128,) * 10, True)])
def test_weights_of_rows_shared_out(dtype, dim, heads, hkv, lens, news, causal):
    # few blocks of keys: their rows go to several workgroups, twice the same bits and with attention on the same workspace in between;
    # many short prompts: more sequences and heads than that is done for
    c = Case(dtype, dim, heads, hkv, 64, lens, news, causal=causal, seed=41)
    plan = plan_for(c)
    gpu = on_gpu(c)
    q = c.q.cuda()
    _, lse = plan.forward(q, *gpu)
    runs = []
    for _ in range(3):
        scores = torch.zeros(c.pages, hkv, c.page, device="cuda")
        plan.weights(q, lse, gpu[0], *gpu[2:], scores)
        out, lse_again = plan.forward(q, *gpu)
        runs.append(scores)
        assert torch.equal(lse_again, lse)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    clean = Case(dtype, dim, heads, hkv, 64, lens, news, causal=causal, seed=41, spare=0.0)
    w, off = ref.weights(clean, lse.cpu())
    near(runs[0], w, off, "scores")


def test_weights_of_missing_pages_and_rows_that_saw_nothing():
    c = Case("bf16", 64, 4, 2, 16, (100, 40), (5, 60), seed=21)   # 20 rows of the second see nothing
    c.table[0, 2] = -1
    plan = plan_for(c)
    gpu = on_gpu(c)
    _, lse = plan.forward(c.q.cuda(), *gpu)
    scores = torch.full((c.pages, 2, 16), 0.5, device="cuda")
    plan.weights(c.q.cuda(), lse, gpu[0], *gpu[2:], scores)
    clean = Case("bf16", 64, 4, 2, 16, (100, 40), (5, 60), seed=21, spare=0.0)
    clean.table[0, 2] = -1
    w, off = ref.weights(clean, lse.cpu())
    near(scores, w + 0.5, off + 2.0 ** -24, "scores")


def all_of(c, plan, gpu):
    out, lse = plan.forward(c.q.cuda(), *gpu)
    scores = torch.zeros(c.pages, c.kv_heads, c.page, device="cuda")
    plan.weights(c.q.cuda(), lse, gpu[0], *gpu[2:], scores)
    return out, lse, scores


@pytest.mark.parametrize("lens,news", [((700, 33), (1, 1)), ((900, 40), (500, 40))])
def test_a_window_that_reaches_past_everything(lens, news):
    plain = Case("bf16", 64, 4, 2, 16, lens, news, seed=46)
    gpu = on_gpu(plain)
    want = all_of(plain, plan_for(plain), gpu)
    for window, sinks in ((2 ** 30, 0), (2 ** 30, 2 ** 30), (900, 3), (5, 2 ** 30)):   # (the last: sinks that are everything)
        c = Case("bf16", 64, 4, 2, 16, lens, news, window=window, sinks=sinks, seed=46)
        got = all_of(c, plan_for(c), gpu)
        for x, y in zip(got, want):
            near(x, y.double().cpu(), 2.0 ** -7 * y.double().cpu().abs() + 2.0 ** -20, (window, sinks))


@pytest.mark.parametrize("heads,hkv", [(40, 1), (33, 1), (14, 2), (130, 1)])
@pytest.mark.parametrize("lens,news", [((300, 70), (1, 5)), ((200, 7), (90, 7))])
def test_groups_of_any_size(heads, hkv, lens, news):
    c = Case("fp16", 64, heads, hkv, 32, lens, news, seed=47)
    check_forward(c)
    clean = Case("fp16", 64, heads, hkv, 32, lens, news, seed=47, spare=0.0)
    _, lse, scores = all_of(c, plan_for(c), on_gpu(c))
    w, off = ref.weights(clean, lse.cpu())
    near(scores, w, off, "scores")


def test_as_many_sequences_as_a_call_may_have():
    lens = [1 + (37 * i) % 50 for i in range(4096)]
    news = [(i % 3 != 0) + (i % 512 == 5) * 20 for i in range(4096)]
    news = [min(n, l) for n, l in zip(news, lens)]
    c = Case("bf16", 64, 4, 2, 16, lens, news, seed=48)
    check_forward(c)
    clean = Case("bf16", 64, 4, 2, 16, lens, news, seed=48, spare=0.0)
    plan, gpu = plan_for(c), on_gpu(c)
    _, lse, scores = all_of(c, plan, gpu)
    w, off = ref.weights(clean, lse.cpu())
    near(scores, w, off, "scores")
    # and their eviction to 16 tokens each: those that drew most, in their order
    kept_table = torch.arange(4096, dtype=torch.int32).view(-1, 1) + c.pages
    k = torch.cat([gpu[0], torch.zeros(4096, 2, 16, 64, dtype=gpu[0].dtype, device="cuda")])
    v = torch.cat([gpu[1], torch.zeros(4096, 2, 16, 64, dtype=gpu[1].dtype, device="cuda")])
    scores = torch.cat([scores, torch.zeros(4096, 2, 16, device="cuda")])
    kept, kept_lens = plan.evict(k, v, scores, gpu[2], gpu[3], kept_table.cuda(), 16)
    assert kept_lens.tolist() == [min(n, 16) for n in lens]
    flat = scores.cpu()
    for b in range(0, 4096, 37):
        pages = c.table[b]
        for g in range(2):
            mine = torch.tensor([flat[pages[j // 16], g, j % 16].item() for j in range(lens[b])])
            best = sorted(sorted(range(lens[b]), key=lambda j: (-mine[j].item(), j))[:16])
            assert [x for x in kept[b, g].tolist() if x >= 0] == best, (b, g)


def fill_scores(c, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(c.pages, c.kv_heads, c.page, generator=g)
    if kind == "ties":
        return (x * 2).round().abs()
    if kind == "zeros":
        return torch.where(x > 2, x, torch.where(x > 0, 0.0, -0.0))
    if kind == "odd":
        x = torch.where(x > 1.5, math.inf, x)
        x = torch.where(x < -1.5, math.nan, x)
        return torch.where((x > -1.5) & (x < -1.2), -math.inf, x)
    if kind == "tiny":   # the lowest bits decide
        return 1 + torch.randint(0, 50, x.shape, generator=g) * 2.0 ** -23
    return torch.exp(3 * x)


@pytest.mark.parametrize("kind", ["exp", "ties", "zeros", "odd", "tiny"])
@pytest.mark.parametrize("lens,budget,first,last", [((1, 40, 41, 300), 40, 0, 0), ((90, 260, 17), 33, 3, 7), ((500,), 20, 20, 0), ((500, 12), 20, 5, 15),
                                                    ((2500, 1100), 1030, 4, 100), ((70,), 1, 0, 0), ((70,), 1, 0, 1), ((0, 130), 64, 1, 1)])
def test_evict(kind, lens, budget, first, last):
    page, hkv = 16, 3
    c = Case("bf16", 64, 3, hkv, page, lens, (0,) * len(lens), seed=22, spare=0.0)
    if len(lens) > 1:
        c.table[-1, 1] = -1   # tokens whose page is not there
    scores = fill_scores(c, kind, 23)
    kept_pages = -(-budget // page)
    B = len(lens)
    pages = c.pages + B * kept_pages
    kept_table = torch.randperm(B * kept_pages, generator=torch.Generator().manual_seed(24)).reshape(B, -1).int() + c.pages
    k, v = (torch.cat([x, torch.full((pages - c.pages, hkv, page, 64), 9.0).to(x.dtype)]) for x in (c.k, c.v))
    s = torch.cat([scores, torch.full((pages - c.pages, hkv, page), 9.0)])
    plan = plan_for(c)
    gk, gv, gs = k.cuda(), v.cuda(), s.cuda()
    kept, kept_lens = plan.evict(gk, gv, gs, c.table.cuda(), c.kv_lens().cuda(), kept_table.cuda(), budget, first, last)
    torch.cuda.synchronize()
    assert kept_lens.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        at = torch.tensor([-1 if c.row(b, j) is None else c.row(b, j) for j in range(n)], dtype=torch.long)
        there = at >= 0
        for h in range(hkv):
            x = scores[at.clamp(min=0), h, torch.arange(n) % page]
            places = ref.kept(x, there, budget, first, last)
            assert kept[b, h].tolist() == places + [-1] * (budget - len(places)), (b, h)
            for i, j in enumerate(places):
                to, row = int(kept_table[b, i // page]), i % page
                if there[j]:
                    k[to, h, row], v[to, h, row], s[to, h, row] = k[at[j], h, j % page], v[at[j], h, j % page], s[at[j], h, j % page]
    assert torch.equal(gk.cpu(), k) and torch.equal(gv.cpu(), v) and torch.equal(gs.cpu().view(torch.int32), s.view(torch.int32))


@pytest.mark.parametrize("kind", ["exp", "ties", "zeros", "odd", "tiny"])
@pytest.mark.parametrize("lens,budget,first,last,heads", [((21000, 30001), 5000, 4, 100, 1), ((9000, 70), 60, 3, 7, 4), ((40000,), 39999, 0, 0, 2),
                                                          ((33333, 9, 8200), 8192, 0, 8190, 2), ((12345,), 10, 5, 5, 1)])
def test_evict_of_long_sequences(kind, lens, budget, first, last, heads):
    """Selections that several workgroups share."""
    page = 64
    c = Case("bf16", 64, heads, heads, page, (0,) * len(lens), (0,) * len(lens), spare=0.0)
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(31)).int()
    c.lens, c.pages = list(lens), sum(need)
    c.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        c.table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
    c.table[0, 17] = c.pages + 10 ** 6
    kept_pages = -(-budget // page)
    pages = c.pages + len(lens) * kept_pages
    kept_table = (torch.arange(len(lens) * kept_pages, dtype=torch.int32) + c.pages).reshape(len(lens), -1)
    k = torch.randn(pages, heads, page, 64, device="cuda").bfloat16()
    v, scores = torch.randn_like(k), fill_scores(c, kind, 32)
    s = torch.cat([scores, torch.zeros(pages - c.pages, heads, page)]).cuda()
    k2, v2, s2 = k.clone(), v.clone(), s.clone()
    kept, kept_lens = plan_for(c).evict(k, v, s, c.table.cuda(), c.kv_lens().cuda(), kept_table.cuda(), budget, first, last)
    for b, n in enumerate(lens):
        at = torch.tensor([-1 if c.row(b, j) is None else c.row(b, j) for j in range(n)], dtype=torch.long)
        for h in range(heads):
            places = ref.kept(scores[at.clamp(min=0), h, torch.arange(n) % page], at >= 0, budget, first, last)
            assert kept[b, h].tolist() == places + [-1] * (budget - len(places)), (b, h)
            i, j = torch.arange(len(places)), torch.tensor(places)
            i, j = i[at[j] >= 0], j[at[j] >= 0]
            to, row = kept_table[b].long()[i // page], i % page
            for x in (k2, v2, s2):
                x[to, h, row] = x[at[j], h, j % page]
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(s.view(torch.int32), s2.view(torch.int32))


@pytest.mark.parametrize("page", [16, 64])
def test_append(page):
    c = Case("fp16", 128, 4, 2, page, (40, 0, 17, 300, 5), (7, 0, 1, 130, 5), seed=25, spare=0.0, extra_rows=4)
    c.table[3, 170 // page + 1] = -1
    plan = plan_for(c)
    g = torch.Generator().manual_seed(26)
    new_k, new_v = (torch.randn(c.tokens, 2, 128, generator=g).half() for _ in range(2))
    for by_head in (False, True):
        k, v, s = c.k.clone(), c.v.clone(), torch.ones(c.pages, 2, page)
        gk, gv, gs = k.cuda(), v.cuda(), s.cuda()
        nk, nv = ((x.transpose(0, 1).contiguous().transpose(0, 1) if by_head else x).cuda() for x in (new_k, new_v))
        plan.append(nk, nv, gk, gv, c.table.cuda(), c.kv_lens().cuda(), c.starts.cuda(), gs)
        for b in range(5):
            for i in range(c.news[b]):
                j = c.lens[b] - c.news[b] + i
                p = c.row(b, j)
                if p is not None:
                    k[p, :, j % page], v[p, :, j % page], s[p, :, j % page] = new_k[c.starts[b] + i], new_v[c.starts[b] + i], 0
        assert torch.equal(gk.cpu(), k) and torch.equal(gv.cpu(), v) and torch.equal(gs.cpu(), s)


def test_a_serving_loop():
    """Prompts in, tokens one by one, the cache shrunk in between: every step against the definition over the rows that should be there."""
    heads, hkv, d, page, budget, dtype = 4, 2, 64, 16, 48, "bf16"
    B, prompts = 3, [70, 33, 5]
    g = torch.Generator().manual_seed(27)
    pages = 64
    k, v = (torch.full((pages, hkv, page, d), float("nan"), dtype=TORCH[dtype], device="cuda") for _ in range(2))
    scores = torch.full((pages, hkv, page), float("nan"), device="cuda")
    tables = [torch.arange(B * 8, dtype=torch.int32).reshape(B, 8), torch.arange(B * 8, 2 * B * 8, dtype=torch.int32).reshape(B, 8)]
    plan = paged.PagedAttention(heads, d, kv_heads=hkv, dtype=dtype, page_size=page, max_batch=B, max_tokens=sum(prompts))
    held_k, held_v = ([[torch.zeros(0, d, dtype=TORCH[dtype]) for _ in range(hkv)] for _ in range(B)] for _ in range(2))
    drawn = [[torch.zeros(0, dtype=torch.float64) for _ in range(hkv)] for _ in range(B)]
    lens = [0] * B
    at = 0
    for step in range(12):
        news = prompts if step == 0 else [1, 2, 1]
        lens = [n + m for n, m in zip(lens, news)]
        starts = [sum(news[:b]) for b in range(B + 1)]
        T = sum(news)
        q, nk, nv = (torch.randn(T, h, d, generator=g).to(TORCH[dtype]) for h in (heads, hkv, hkv))
        args = (tables[at].cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda())
        plan.append(nk.cuda(), nv.cuda(), k, v, *args, scores)
        out, lse = plan.forward(q.cuda(), k, v, *args)
        plan.weights(q.cuda(), lse, k, *args, scores)
        for b in range(B):
            t = slice(starts[b], starts[b + 1])
            for h in range(hkv):
                held_k[b][h], held_v[b][h] = torch.cat([held_k[b][h], nk[t, h]]), torch.cat([held_v[b][h], nv[t, h]])
                drawn[b][h] = torch.cat([drawn[b][h], torch.zeros(news[b], dtype=torch.float64)])
                n, L = news[b], lens[b]
                mask = torch.arange(L)[None, :] > (L - n + torch.arange(n))[:, None]
                for x in range(h * 2, h * 2 + 2):
                    s = (q[t, x].double() @ held_k[b][h].double().T / 8).masked_fill(mask, -math.inf)
                    p = torch.softmax(s, dim=1)
                    o = p @ held_v[b][h].double()
                    # (2^-8: half a step of bf16, once for the probabilities and once for the result)
                    assert ((out[t, x].double().cpu() - o).abs() <= 2.0 ** -8 * (o.abs() + 1.01 * (p @ held_v[b][h].double().abs()))).all(), (step, b, x)
                    drawn[b][h] += p.sum(dim=0)
                got = torch.stack([scores[int(tables[at][b, j // page]), h, j % page] for j in range(L)]).double().cpu()
                assert ((got - drawn[b][h]).abs() <= 1e-4 * drawn[b][h] + 1e-6).all(), (step, b, h)
        if step in (3, 7):
            kept, kept_lens = plan.evict(k, v, scores, *args[:2], tables[1 - at].cuda(), budget, 2, 8)
            at = 1 - at
            lens = kept_lens.tolist()
            for b in range(B):
                for h in range(hkv):
                    stay = [j for j in kept[b, h].tolist() if j >= 0]
                    assert len(stay) == lens[b]
                    # which tokens these are goes by the kernel's own sums (two that drew the same to the last bit may change places)
                    held_k[b][h], held_v[b][h], drawn[b][h] = held_k[b][h][stay], held_v[b][h][stay], drawn[b][h][stay]


def test_captured_calls_of_long_and_short_sequences():
    """One graph, replayed with lengths that go every way: parts in two steps, row tiles of a wave's own, shares of many rows, rows of a block of
    keys in parts -- and nothing at all; another plan's eager calls on the same workspace in between."""
    heads, hkv, page, d, B, T, cap = 8, 1, 64, 64, 300, 800, 9000
    g = torch.Generator().manual_seed(49)
    pages = cap // page + 1
    k, v = (torch.randn(2 * pages, hkv, page, d, generator=g).half().cuda() for _ in range(2))
    table = torch.randint(0, 2 * pages, (B, pages), generator=g, dtype=torch.int32).cuda()   # (read only: shared as it falls)
    q = torch.randn(T, heads, d, generator=g).half().cuda()
    lens, starts = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    room = torch.zeros(paged.PagedAttention(heads, d, kv_heads=hkv, max_batch=B, max_tokens=T).workspace_bytes(), dtype=torch.uint8, device="cuda")
    made = dict(kv_heads=hkv, max_batch=B, max_tokens=T, workspace=(room.data_ptr(), room.numel()))
    plan, other = paged.PagedAttention(heads, d, **made), paged.PagedAttention(heads, d, **made)
    apart = paged.PagedAttention(heads, d, kv_heads=hkv, max_batch=B, max_tokens=T)
    out, lse = torch.zeros_like(q), torch.zeros(heads, T, device="cuda")
    own = torch.arange(2 * pages, dtype=torch.int32, device="cuda").view(2, pages)    # for the weights: no page twice
    scores = torch.zeros(2 * pages, hkv, page, device="cuda")

    def step(plan, out, lse, scores):
        plan.forward(q, k, v, table, lens, starts, out=out, lse=lse)
        plan.weights(q, lse, k, own, lens[:2], starts[:3], scores)

    step(plan, out, lse, scores)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(plan, out, lse, scores)
    for L, n in (([9000, 1], [1, 1]), ([5, 7], [1, 1]), ([9000, 8700], [300, 200]), ([1 + i % 60 for i in range(B)], [1] * B), ([], []), ([900, 8000], [600, 1]),
                 ([9000, 1], [1, 1])):
        L, n = L + [0] * (B - len(L)), n + [0] * (B - len(n))
        lens.copy_(torch.tensor(L, dtype=torch.int32))
        starts.copy_(torch.tensor([sum(n[:i]) for i in range(B + 1)], dtype=torch.int32))
        want = [torch.zeros_like(x) for x in (out, lse, scores)]
        step(apart, *want)
        for x in (out, lse, scores):
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((out, lse, scores), want)), L[:3]
        got = [torch.zeros_like(x) for x in want]
        step(other, *got)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), L[:3]


def test_captured_calls_follow_the_lengths_on_the_device():
    """append, forward, weights and evict in one graph, replayed with other lengths, tokens and tables, with eager work in between."""
    heads, hkv, d, page, B = 8, 2, 128, 16, 4
    g = torch.Generator().manual_seed(28)
    pages, cap = 160, 16
    base_k, base_v = (torch.randn(pages, hkv, page, d, generator=g).bfloat16().cuda() for _ in range(2))
    k, v, scores = base_k.clone(), base_v.clone(), torch.zeros(pages, hkv, page, device="cuda")
    T = 40
    q, nk, nv = (torch.randn(T, h, d, generator=g).bfloat16().cuda() for h in (heads, hkv, hkv))
    table, lens, starts = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((B, cap), (B,), (B + 1,)))
    kept_table = torch.arange(pages - B * 4, pages, dtype=torch.int32, device="cuda").reshape(B, 4)
    plan = paged.PagedAttention(heads, d, kv_heads=hkv, dtype="bf16", page_size=page, max_batch=B, max_tokens=T, window=100, sinks=4)
    out, lse = torch.zeros_like(q), torch.zeros(heads, T, device="cuda")
    kept, kept_lens = torch.zeros(B, hkv, 60, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(stream=None):
        plan.append(nk, nv, k, v, table, lens, starts, scores, stream=stream)
        plan.forward(q, k, v, table, lens, starts, out, lse, stream=stream)
        plan.weights(q, lse, k, table, lens, starts, scores, stream=stream)
        plan.evict(k, v, scores, table, lens, kept_table, 60, 4, 8, kept, kept_lens, stream=stream)

    def fresh():
        k.copy_(base_k), v.copy_(base_v), scores.zero_(), out.zero_(), lse.zero_(), kept.zero_(), kept_lens.zero_()

    step()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side)
    for i, (ls, ns) in enumerate([([1, 50, 250, 33], [1, 1, 1, 1]), ([200, 0, 31, 256], [13, 0, 20, 7]), ([40, 40, 40, 40], [40, 0, 0, 0]), ([3, 256, 9, 100], [0, 40, 0, 0])]):
        perm = torch.randperm(pages - B * 4, generator=g)[:B * cap].reshape(B, cap).int()
        table.copy_(perm), lens.copy_(torch.tensor(ls, dtype=torch.int32)), starts.copy_(torch.tensor([sum(ns[:b]) for b in range(B + 1)], dtype=torch.int32))
        q.copy_(torch.randn(T, heads, d, generator=g))
        fresh()
        step()
        torch.cuda.synchronize()
        eager = [x.clone() for x in (k, v, scores, out, lse, kept, kept_lens)]
        fresh()
        (base_k.float().sum() + 1).item()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((k, v, scores, out, lse, kept, kept_lens), eager):
            assert torch.equal(x, y), i


def test_calls_on_another_stream_and_plans_side_by_side():
    cases = [Case("bf16", 128, 8, 2, 16, (900, 333), (1, 1), seed=29), Case("fp16", 64, 4, 4, 32, (600,), (200,), seed=30)]
    plans, states, expected = [], [], []
    for c in cases:
        plans.append(plan_for(c))
        states.append((c.q.cuda(), *on_gpu(c)))
        expected.append(plans[-1].forward(*states[-1]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = [p.forward(*s, stream=t) for p, s, t in zip(plans, states, streams)]
        for t in streams:
            t.synchronize()
        for x, y in zip(got, expected):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_the_general_way_of_a_call_does_the_same():
    """Calls are checked and made by ringattn_calls where everything is as expected; without it the same launches are made."""
    c = Case("bf16", 64, 4, 2, 16, (61, 333, 0), (1, 140, 0), seed=34, spare=0.0)
    g = torch.Generator().manual_seed(35)
    new_k, new_v = (torch.randn(c.tokens, 2, 64, generator=g).bfloat16().cuda() for _ in range(2))
    kept_table = torch.arange(c.pages - 2, c.pages, dtype=torch.int32).repeat(3, 1).cuda()[:, :2].contiguous()
    results = []
    for native in (True, False):
        plan = plan_for(c)
        if not native:
            plan._call_type = None
        k, v, table, lens, starts = on_gpu(c)
        q = c.q.cuda()
        scores = torch.zeros(c.pages, 2, 16, device="cuda")
        plan.append(new_k, new_v, k, v, table, lens, starts, scores)
        out, lse = torch.zeros_like(q), torch.zeros(4, c.tokens, device="cuda")
        plan.forward(q, k, v, table, lens, starts, out, lse)
        plan.weights(q, lse, k, table, lens, starts, scores)
        kept, kept_lens = torch.zeros(3, 2, 20, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
        plan.evict(k[:, :, :], v, scores, table, lens, kept_table, 20, 2, 3, kept, kept_lens)
        results.append((k[:-2], v[:-2], out, lse, scores[:-2], kept, kept_lens))
        assert bool(plan._native) == native
    for x, y in zip(*results):
        assert torch.equal(x, y)
    for bad in (q[:, :3], q.float(), q.cpu(), q.transpose(1, 2)):   # refused as the general way refuses them
        with pytest.raises(ValueError):
            plan_for(c).forward(bad, k, v, table, lens, starts, out, lse)
    with pytest.raises(ValueError):
        plan_for(c).weights(q, lse, k, table, lens, starts, scores.double())
    plan = plan_for(c)
    plan.append(new_k, new_v, k, v, table, lens, starts)
    plan.close()
    with pytest.raises(Exception, match="plan"):
        plan.append(new_k, new_v, k, v, table, lens, starts)


def test_nothing_to_do():
    plan = paged.PagedAttention(4, 64, kv_heads=2, dtype="fp16", page_size=16, max_batch=2, max_tokens=4)
    k = torch.zeros(3, 2, 16, 64, dtype=torch.float16, device="cuda")
    none = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    table, lens, starts = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((0, 2), (0,), (1,)))
    out, lse = plan.forward(none, k, k, table, lens, starts)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    plan.append(none[:, :2], none[:, :2], k, k, table, lens, starts)
    table, lens, starts = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((2, 2), (2,), (3,)))
    plan.forward(none, k, k, table, lens, starts)
