"""Shaped scores over the paged cache where the work is dealt out otherwise than in small calls: row tiles with hundreds of key tiles, whose pages are
held 64 tiles at a time; shares of several sizes; launches without shares; batches of more sequences than a wave has lanes."""
import math

import pytest
import torch

import scored_reference as ref
import scored_samples as samples
from test_gpu_paged_scored import check, compare, docs_of, plan_of, sequences, slopes_of

pytestmark = pytest.mark.gpu


def dealt(c, few_most):
    """(key tiles a share is to have, [(row tiles, key tiles, shares a row tile)] of the sequences of more than few_most rows), as find_place works it out
    for a call whose row tiles may be cut and whose documents, if any, begin with the first new token's."""
    group, tiles = c.heads // c.kv_heads, []
    for b, (L, n) in enumerate(zip(c.lens, c.news)):
        if n * group <= few_most:
            continue
        first = min(c.first[int(c.starts[b])], L - n) if c.first is not None else 0
        tiles.append((-(-n * group // 256), -(-L // 32) - first // 32))
    share = max(sum(t * k for t, k in tiles) * c.kv_heads / 256, 8)
    made = []
    for t, k in tiles:
        s = max(1, math.floor(k / share + 0.01)) if share > 8 else -(-k // 8)
        made.append((t, k, s if k - -(-k // s) >= 12 else 1))
    return share, made


def check_all(c):
    """All rows and all keys.  Each weight below 2^-126 is 0: a sum is off by as many of them as it has terms at most."""
    out, lse = check(c, do_weights=False)
    plan = plan_of(c)
    slopes, prefix, first = c.given()
    scores = plan.weights(c.q.cuda(), lse, c.k.cuda(), *sequences(c), torch.zeros(c.pages, c.kv_heads, c.page, device="cuda"), prefix_lens=prefix, first_keys=first)
    want, tol = ref.weights(c, lse.cpu())
    compare(scores, want, tol + max(c.news) * (c.heads // c.kv_heads) * 2.0 ** -126, "weights")
    return out, lse


def check_some(c, heads, step, weights=True, same=True):
    """The heads `heads`, every step-th new token and the first and last of every sequence, the weights of keys from all over."""
    plan = plan_of(c)
    slopes, prefix, first = c.given()
    q, k, v = c.q.cuda(), c.k.cuda(), c.v.cuda()
    out, lse = plan.forward(q, k, v, *sequences(c), prefix_lens=prefix, first_keys=first)
    if same:
        again = plan.forward(q, k, v, *sequences(c), prefix_lens=prefix, first_keys=first)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    for b, n in enumerate(c.news):
        if not n:
            continue
        idx = torch.tensor(sorted({0, n - 1, n // 2} | set(range(5 % n, n, step))))
        at = int(c.starts[b]) + idx
        for h in heads:
            o, z, tol, tol_z = samples.rows(c, b, h, idx)
            compare(out.cpu()[at, h], o, tol, ("out", b, h))
            compare(lse.cpu()[h, at], z, tol_z, ("lse", b, h))
    if weights:
        scores = plan.weights(q, lse, k, *sequences(c), torch.zeros(c.pages, c.kv_heads, c.page, device="cuda"), prefix_lens=prefix, first_keys=first).cpu()
        for b, L in enumerate(c.lens):
            if not c.news[b]:
                continue
            keys = torch.tensor(sorted({0, L - 1, L // 2} | set(range(3 % L, L, max(1, L // 40)))))
            for g in {h // (c.heads // c.kv_heads) for h in heads}:
                w, tol = samples.weights(c, b, g, keys, lse.cpu())
                there = [i for i, j in enumerate(keys.tolist()) if c.row(b, j) is not None]
                got = torch.stack([scores[c.row(b, int(keys[i])), g, int(keys[i]) % c.page] for i in there])
                compare(got, w[there], tol[there], ("weights", b, g))
    return out, lse


L, N = 8229, 1100
LONG = dict(lens=[L], news=[N], heads=32, kv_heads=4, dim=64, page=64)
BORDERS = [500] * 613 + [6000] * 200 + [L - 250] * (N - 813)   # documents that begin before the chunk, far in it, and within it


@pytest.mark.parametrize("kind,dtype,dim", [("cap", "bf16", 64), ("cap", "fp16", 128), ("slopes", "bf16", 64), ("all", "bf16", 64), ("all", "fp16", 128), ("documents", "bf16", 128),
                                            ("window", "fp16", 64)])
def test_hundreds_of_key_tiles_a_workgroup(kind, dtype, dim):
    """A chunk whose row tiles have some 240 key tiles each, pages missing in the first, the second and the last 64 of them."""
    more = {"cap": dict(cap=20.0), "slopes": dict(slopes=slopes_of(32)), "all": dict(cap=7.0, slopes=[s / 16 for s in slopes_of(32)], first=BORDERS, prefix=[40]),
            "documents": dict(first=BORDERS), "window": dict(window=7000, sinks=70, cap=30.0)}[kind]
    c = ref.Case(**dict(LONG, dtype=dtype, dim=dim), seed=len(kind), **more)
    for entry in (9, 46, 100, 128):
        c.table[0, entry] = -1
    share, made = dealt(c, 128)
    assert share > 128 and made[0][2] == 1 and made[0][1] > 192
    check_some(c, (0, 7, 13, 31), 97)


@pytest.mark.parametrize("kind", ["all", "slopes", "documents"])
def test_shares_of_a_long_sequence_beside_a_short_one(kind):
    """More to do than workgroups that run at once, and a sequence whose row tiles are cut all the same."""
    lens, news = [6000, 1500, 800], [40, 700, 1]
    more = {"all": dict(cap=9.0, slopes=[s / 8 for s in slopes_of(16)], prefix=[30, 0, 5]), "slopes": dict(slopes=slopes_of(16)),
            "documents": dict(first=[3] * 25 + [3000] * 15 + docs_of([1500], [700], 450) + [0])}[kind]
    c = ref.Case(lens=lens, news=news, heads=16, kv_heads=2, dim=128, page=32, seed=len(kind), **more)
    share, made = dealt(c, 64)
    assert share > 8 and made[0][2] > 1
    check_some(c, (0, 5, 15), 41)


@pytest.mark.parametrize("kind", ["cap", "all"])
def test_row_tiles_that_fill_the_device_are_not_shared_out(kind):
    """As many row tiles as there are compute units: a launch without shares and without their putting together."""
    c = ref.Case(lens=[3000], news=[2100], heads=32, kv_heads=8, dim=64, page=128, seed=4, cap=12.0,
                 **(dict(slopes=[s / 8 for s in slopes_of(32)], first=docs_of([3000], [2100], 1700), prefix=[64]) if kind == "all" else {}))
    assert 2100 * 4 // 256 * 8 >= 256
    check_some(c, (0, 9, 31), 211)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("kind", ["documents", "window"])
def test_a_hidden_v_that_is_odd_far_into_the_walk(kind, value):
    """In key tile 158, which some rows of every workgroup see and others do not: the walk begins again when it has held its pages for the fourth time."""
    j = 5058
    first = [5500 if i % 3 == 1 else 0 for i in range(N)] if kind == "documents" else None
    more = dict(first=first) if kind == "documents" else dict(window=2600)   # (tokens 7129 to 8228: some see place 5058, later ones do not)
    c = ref.Case(**LONG, seed=3, cap=10.0, **more)
    c.v[c.row(0, j), :, j % 64, 5] = value
    c.table[0, 70] = -1
    assert dealt(c, 128)[0] > 100
    idx = torch.tensor([0, 1, 2, 3, 300, 301, 302, 528, 529, 530, 1097, 1098, 1099])
    plan = plan_of(c)
    out, lse = plan.forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c), first_keys=c.given()[2])
    ok = torch.tensor([first[i] <= j if first else j > L - N + i - 2600 for i in idx.tolist()])
    assert ok.any() and not ok.all()
    for h in (0, 17, 31):
        o, z, tol, tol_z = samples.rows(c, 0, h, idx)
        assert torch.isfinite(o[~ok]).all() and not torch.isfinite(o[ok][:, 5]).any()
        compare(out.cpu()[idx, h], o, tol, ("out", h))
        compare(lse.cpu()[h, idx], z, tol_z, ("lse", h))


def test_open_calls_of_many_rows_with_a_cap():
    """No causality: every row sees every key."""
    check_all(ref.Case(lens=[700, 90], news=[531, 90], heads=4, kv_heads=2, page=64, causal=False, cap=6.0, seed=21))
    check_all(ref.Case(lens=[900], news=[300], heads=4, kv_heads=1, dim=64, dtype="fp16", causal=False, cap=0.5, seed=22))


# ---- more sequences than a wave has lanes
def batch_of(size, chunks, none=()):
    """`size` sequences of some hundred tokens, a new one each; chunks: {sequence: (length, new tokens)}."""
    lens = [chunks[i][0] if i in chunks else (i * 137) % 611 + 1 for i in range(size)]
    news = [chunks[i][1] if i in chunks else 0 if i in none else 1 for i in range(size)]
    return lens, news


MANY_SEQUENCES = {
    "64 tokens": batch_of(64, {}),
    "65 tokens": batch_of(65, {}),
    "65, the last has none": batch_of(65, {}, (64,)),
    "65, the last a chunk": batch_of(65, {64: (2600, 300)}),
    "64 with chunks": batch_of(64, {0: (2600, 300), 63: (700, 200), 30: (90, 90)}),
    "131 with chunks in the second and third look": batch_of(131, {70: (2600, 300), 100: (600, 150), 129: (90, 90), 130: (1500, 40)}, (3, 64, 65, 128)),
}


@pytest.mark.parametrize("kind", ["all", "slopes", "documents"])
@pytest.mark.parametrize("name", MANY_SEQUENCES)
def test_more_sequences_than_lanes(name, kind):
    lens, news = MANY_SEQUENCES[name]
    more = {"all": dict(cap=5.0, slopes=[0.1, 0.02, 0.5, 0.0], prefix=[(i * 29) % 50 for i in range(len(lens))], first=docs_of(lens, news, 77)),
            "slopes": dict(slopes=[0.1, 0.02, 0.5, 0.0], prefix=[(i * 7) % 40 for i in range(len(lens))]), "documents": dict(first=docs_of(lens, news, 301))}[kind]
    c = ref.Case(lens=lens, news=news, heads=4, kv_heads=2, dim=64, page=32, seed=len(lens), **more)
    if "chunk" in name and kind == "slopes":
        share, made = dealt(c, 64)
        assert share == 8 and max(s for _, _, s in made) > 1   # (some are cut, and put together)
    out, lse = check_all(c)
    plan = plan_of(c)
    slopes, prefix, first = c.given()
    again = plan.forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c), prefix_lens=prefix, first_keys=first)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    if kind == "all":
        check_all(ref.Case(lens=lens, news=news, heads=4, kv_heads=2, dim=64, page=32, seed=len(lens), window=90, sinks=5, **more))


def test_long_sequences_of_a_large_batch():
    """70 sequences, one of which is long enough for shares of more than the least."""
    chunks = {66: (9000, 200), 3: (3000, 900), 69: (2000, 2000)}
    lens, news = batch_of(70, chunks)
    c = ref.Case(lens=lens, news=news, heads=8, kv_heads=2, dim=64, page=64, seed=7, cap=11.0, slopes=[s / 8 for s in slopes_of(8)], prefix=[(13 * i) % 90 for i in range(70)])
    share, made = dealt(c, 64)
    assert share > 8 and any(s > 1 for _, _, s in made)
    check_some(c, (0, 6), 173)


# ---- what is hidden, of few rows
@pytest.mark.parametrize("lens,news", [([300], [7]), ([90, 64], [3, 1])])
@pytest.mark.parametrize("which,value", [("k", float("nan")), ("k", float("inf")), ("v", float("inf")), ("v", float("-inf")), ("v", float("nan"))])
def test_hidden_places_of_few_rows(lens, news, which, value):
    """One value of a row of K or V that is no number, in the document in front of that of the last new token."""
    first = docs_of(lens, news, 61)
    b = len(lens) - 1
    j = max(0, first[-1] - 1)
    first[int(sum(news)) - news[b]] = 0   # (the last sequence's first new token sees all)
    if news[b] == 1:
        first[-1] = j + 1
    c = ref.Case(lens=lens, news=news, heads=4, kv_heads=2, first=first, cap=4.0, seed=8)
    for g in range(2):
        (c.k if which == "k" else c.v)[c.row(b, j), g, j % c.page, 9] = value
    out, lse = plan_of(c).forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c), first_keys=c.given()[2])
    of_b = torch.zeros(sum(news), dtype=torch.bool)
    of_b[sum(news) - news[b]:] = True
    sees = of_b & torch.tensor([x <= j for x in first])
    assert not sees.all() and (sees.any() or news[b] == 1)
    if which == "v":
        want, want_lse, tol, tol_lse = ref.attend(c)
        compare(out, want, tol, "out")
        compare(lse, want_lse, tol_lse, "lse")
        assert not sees.any() or not torch.isfinite(want[sees][:, :, 9]).any()
        return
    # (a score of no number makes its row none; an infinite one is a cap)
    clean = ref.Case(lens=lens, news=news, heads=4, kv_heads=2, first=first, cap=4.0, seed=8)
    want, want_lse, tol, tol_lse = ref.attend(clean)
    compare(out[~sees], want[~sees], tol[~sees], "out")
    compare(lse[:, ~sees], want_lse[:, ~sees], tol_lse[:, ~sees], "lse")
    assert out[sees].isnan().all() if math.isnan(value) else torch.isfinite(out[sees]).all()


# ---- how far a cap's scores are off
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("lens,news", [([500], [1]), ([1000], [300])])
def test_a_large_cap_is_off_by_its_last_bits(lens, news, slopes):
    """Scores near 0 under a cap of 1024, whose tanh is nearly its argument.  In units of 2^-24 of the cap a score is off by: 2 of the exponential (2^-23 of e^2y,
    near 1, a quarter of which reaches 1 / (e^2y + 1), which counts twice the cap: 1), the sum e^2y + 1 (half a step of 2, a quarter, twice: 1), the reciprocal (a
    step of 1/2, twice: 2), the argument (2^-23 of itself, at most 0.23 of which: 0.9), the rounded cap (1): 5.9; a slope's sum is rounded where it is the size
    of two caps: 2.  The sum of the weights has a rounding for every key, the LSE those of its size."""
    c = ref.Case(lens=lens, news=news, heads=4, kv_heads=2, dim=64, dtype="fp16", cap=1024.0, slopes=[0.01, 0.0, 0.1, 1e-3] if slopes else None, sigma=0.3, seed=5)
    out, lse = plan_of(c).forward(c.q.cuda(), c.k.cuda(), c.v.cuda(), *sequences(c))
    for h in range(4):
        k, there = c.rows(c.k, 0, h // 2)
        ok, x, _ = c.scores(0, h, k, there)
        _, far = c.sight(0, there)
        q = c.q[:, h].double()
        off = (c.dim + 4) * (q.abs() @ k.abs().T * c.scale) + (8 if slopes else 6) * 1024 + (4 * c.slopes[h] * far.double() if slopes else 0) + 4
        z = torch.logsumexp(x, dim=1)
        p = torch.where(ok, torch.exp(x - z[:, None]), 0.0)
        tol = (p * off).sum(dim=1) * 2.0 ** -24 + (ok.sum(dim=1) + 8) * 2.0 ** -24 + 2.0 ** -22 * (1 + z.abs())
        assert tol.max() < (2 if slopes else 1.5) * 2.0 ** -22 * 1024 + 2.0 ** -11
        compare(lse[h], z, tol, ("lse", h))
