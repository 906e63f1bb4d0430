"""Shaped scores over the paged cache: calls that the documentation allows besides those of the other files -- graphs of one plan in turn, partials, as many
sequences as a plan takes, more new tokens than there are, groups of any size, padded rows, another stream."""
import pytest
import torch

import paged_reference
import scored_reference as ref
from test_gpu_paged_scored import compare, docs_of, plan_of, sequences, slopes_of
from test_gpu_paged_scored_long import batch_of, check_all

pytestmark = pytest.mark.gpu


def call(c, plan, **more):
    """(out, lse, scores) of forward and weights."""
    slopes, prefix, first = c.given()
    q, k, v = c.q.cuda(), c.k.cuda(), c.v.cuda()
    out, lse = plan.forward(q, k, v, *sequences(c), prefix_lens=prefix, first_keys=first, **more)
    return out, lse, plan.weights(q, lse, k, *sequences(c), torch.zeros(c.pages, c.kv_heads, c.page, device="cuda"), prefix_lens=prefix, first_keys=first, **more)


def test_graphs_of_one_plan_in_turn():
    """Calls whose row tiles are cut in different ways, of few rows and of many, captured on one workspace and replayed in any order, with eager calls between."""
    heads = dict(heads=4, kv_heads=2, dim=64, page=32, cap=9.0, slopes=[0.1, 0.02, 0.5, 0.0])
    shapes = [([2600, 90], [300, 90]), ([5000], [1]), batch_of(70, {66: (2000, 300)}), ([700] * 5, [40] * 5)]
    cases = [ref.Case(lens=l, news=n, seed=i, prefix=[(9 * j) % 50 for j in range(len(l))], first=docs_of(l, n, 400), **heads) for i, (l, n) in enumerate(shapes)]
    big = max(cases, key=lambda c: c.tokens)
    big_batch = max(len(c.lens) for c in cases)
    from ringattention_amd import paged
    plan = paged.PagedAttention(4, 64, kv_heads=2, dtype="bf16", page_size=32, max_batch=big_batch, max_tokens=big.tokens, softcap=9.0, slopes=big.given()[0])
    graphs, wants, kept = [], [], []
    for c in cases:
        wants.append([x.clone() for x in call(c, plan)])
        slopes, prefix, first = c.given()
        q, k, v, seqs = c.q.cuda(), c.k.cuda(), c.v.cuda(), sequences(c)
        out, lse, scores = torch.zeros_like(q), torch.zeros(4, c.tokens, device="cuda"), torch.zeros(c.pages, 2, 32, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plan.forward(q, k, v, *seqs, out, lse, prefix_lens=prefix, first_keys=first)
            plan.weights(q, lse, k, *seqs, scores, prefix_lens=prefix, first_keys=first)
        graphs.append(g)
        kept.append((q, k, v, seqs, prefix, first, out, lse, scores))
    for turn in range(3):
        for i in (0, 1, 2, 3, 1, 0, 3, 2):
            out, lse, scores = kept[i][-3:]
            for x in (out, lse, scores):
                x.zero_()
            graphs[i].replay()
            if (turn + i) % 2:
                call(cases[(i + 1) % 4], plan)
            torch.cuda.synchronize()
            for got, want in zip((out, lse, scores), wants[i]):
                assert torch.equal(got, want), (turn, i)


@pytest.mark.parametrize("lens,news", [([700, 90], [531, 90]), ([2600, 40], [1, 1]), ([3000], [300])])
def test_partials(lens, news):
    """O in 32 bits, under slopes, prefixes and documents."""
    c = ref.Case(lens=lens, news=news, heads=4, kv_heads=2, dim=128, cap=4.0, slopes=slopes_of(4), prefix=[13] * len(lens), first=docs_of(lens, news, 150), seed=3)
    out, lse, scores = call(c, plan_of(c, partials=True))
    assert out.dtype == torch.float32
    want, want_lse, tol, tol_lse = ref.attend(c)
    compare(out, want, tol, "out")
    compare(lse, want_lse, tol_lse, "lse")


def test_as_many_sequences_as_a_plan_takes():
    lens, news = batch_of(4096, {4000: (300, 9)})
    lens = [n % 97 + 1 if n != 300 else n for n in lens]
    c = ref.Case(lens=lens, news=news, heads=1, kv_heads=1, dim=64, page=64, cap=3.0, slopes=[0.05], prefix=[i % 31 for i in range(4096)], first=docs_of(lens, news, 41), seed=4)
    check_all(c)


@pytest.mark.parametrize("scores", ["slopes", "all"])
@pytest.mark.parametrize("lens,news", [([100], [400]), ([3, 90, 0], [300, 200, 100])])
def test_many_more_new_tokens_than_there_are(lens, news, scores):
    """Tokens at places in front of the first: they see a prefix, or nothing."""
    more = dict(slopes=slopes_of(4), prefix=[37, 60, 0][:len(lens)])
    if scores == "all":
        more.update(cap=6.0, first=[(7 * i) % 50 for i in range(sum(news))], window=40, sinks=2)
    check_all(ref.Case(lens=lens, news=news, heads=4, kv_heads=1, dim=64, seed=5, **more))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (32, 1), (7, 1), (10, 2), (9, 9)])
def test_groups_of_any_size(heads, kv_heads):
    lens, news = [400, 33, 70], [150, 1, 20]
    for more in (dict(cap=5.0, slopes=slopes_of(heads), prefix=[20, 3, 0]), dict(first=docs_of(lens, news, 47) + [0] * 5, window=60, sinks=3)):
        check_all(ref.Case(lens=lens, news=news, heads=heads, kv_heads=kv_heads, dim=64, dtype="fp16", page=16, seed=heads, extra_rows=5, **more))


@pytest.mark.parametrize("page", [16, 1024])
def test_pages_of_the_smallest_and_largest_size(page):
    lens, news = [1500, 1025, 1], [300, 1, 1]
    check_all(ref.Case(lens=lens, news=news, heads=4, kv_heads=2, dim=128, page=page, cap=8.0, slopes=slopes_of(4), prefix=[1030, 16, 1], first=docs_of(lens, news, 1024), seed=page))


def test_another_stream():
    """Both calls, and what they allocate."""
    c = ref.Case(lens=[900, 40], news=[200, 1], heads=4, kv_heads=2, cap=5.0, slopes=slopes_of(4), seed=9)
    plan = plan_of(c)
    want = call(c, plan)
    stream = torch.cuda.Stream()
    slopes, prefix, first = c.given()
    q, k, v, seqs = c.q.cuda(), c.k.cuda(), c.v.cuda(), sequences(c)
    scores = torch.zeros(c.pages, 2, 16, device="cuda")
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        out, lse = plan.forward(q, k, v, *seqs, stream=stream)
    plan.weights(q, lse, k, *seqs, scores, stream=stream)
    stream.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(scores, want[2])


def test_masks_that_hide_nothing_are_the_plain_definition():
    """A window that reaches everything, documents that begin in front, prefixes of nothing, slopes of 0."""
    c = ref.Case(lens=[600, 65], news=[280, 3], heads=4, kv_heads=2, window=5000, slopes=[0.0] * 4, prefix=[0, -3], first=[-5] * 283, seed=2)
    plain = paged_reference.Case(lens=[600, 65], news=[280, 3], heads=4, kv_heads=2, seed=2)
    out, lse, _ = call(c, plan_of(c))
    want, want_lse, tol, tol_lse = paged_reference.attend(plain)
    compare(out, want, 2 * tol, "out")
    compare(lse, want_lse, 2 * tol_lse, "lse")


class Steep(ref.Case):
    """With what the product of a slope and a place is off by besides: the place is that of a lane's first key of a tile, up to 27 further from the row than
    the key itself, and 2^-24 of the product is rounded away, also where the key is the row's own."""

    def scores(self, b, h, k, there):
        ok, s, off = super().scores(b, h, k, there)
        return ok, s, torch.where(ok, off + 28 * abs(self.slopes[h]) * 2.0 ** -24, 0.0)


@pytest.mark.parametrize("prefix,cap", [(False, 0.0), (True, 0.0), (False, 6.0)])
@pytest.mark.parametrize("lens,news", [([50, 301, 64], [1, 1, 1]), ([200, 40], [17, 40]), ([600], [420])])
def test_slopes_of_thousands(lens, news, prefix, cap):
    """One key takes a row: its own, or of negative slopes the farthest."""
    c = Steep(lens=lens, news=news, heads=4, kv_heads=2, dim=64, dtype="fp16", page=32, slopes=[1000.0, -300.0, 37.5, 4096.0], cap=cap,
              prefix=[45, 30, 64][:len(lens)] if prefix else None, seed=21)
    check_all(c)
