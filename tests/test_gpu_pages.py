"""Pages of a cache on the GPU against the definition in pages_reference: whole numbers and copies, so that everything is equal."""
import random

import pytest
import torch

from pages_reference import Pages, entries
from ringattention_amd import paged

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Both:
    """A pool on the device beside its definition; a row of a page's K holds the page's own history of copies."""

    def __init__(self, pages, rows, table_pages, page=16, heads=2, dim=64, seed=0, scores=True, layout="plain"):
        self.want = Pages(pages, rows, table_pages, page)
        self.pool = paged.PagePool(pages, rows, table_pages, page)
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape = (pages, heads, page, dim)
        self.k, self.v = (torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        if layout == "token":    # [pages, page, heads, dim + room]
            def moved(x):
                wide = torch.zeros(pages, page, heads, dim + 8, dtype=x.dtype, device="cuda")
                y = wide[..., :dim].permute(0, 2, 1, 3)
                y.copy_(x)
                return y
            self.k, self.v = moved(self.k), moved(self.v)
        self.scores = torch.randn(shape[:3], generator=g, device="cuda") if scores else None
        self.copies = [x.clone() for x in (self.k, self.v, self.scores) if x is not None]

    def moved(self, pairs):
        if pairs:
            a, b = (torch.tensor(x, device="cuda") for x in zip(*pairs))
            for x in self.copies:
                x[b] = x[a]

    def check(self, what):
        torch.cuda.synchronize()
        p, w = self.pool, self.want
        assert p.lens.tolist() == w.lens, what
        assert p.page_table.tolist() == w.table, what
        assert p.refs.tolist() == w.refs, what
        for got, want in zip([x for x in (self.k, self.v, self.scores) if x is not None], self.copies):
            assert torch.equal(got, want), what

    def update(self, parents=None, add=None, **more):
        short, copies = self.want.update(parents, add)
        self.moved(copies)
        got = self.pool.update(self.k, self.v, ints(parents) if parents is not None else None, ints(add) if add is not None else None, scores=self.scores, **more)
        self.check((parents, add))
        assert got.tolist() == short

    def compact(self):
        n, moves, places = self.want.compact()
        self.moved(moves)
        moved = torch.full((self.want.pages,), -7, dtype=torch.int32, device="cuda")
        got = self.pool.compact(self.k, self.v, scores=self.scores, moved=moved)
        self.check("compact")
        assert got.tolist() == [n] and moved.tolist() == places


@pytest.mark.parametrize("seed", range(12))
def test_any_steps(seed):
    rng = random.Random(seed)
    page = rng.choice((16, 32, 64))
    rows = rng.choice((1, 2, 5, 40, 70))
    b = Both(rng.choice((3, 17, 200, 1001)), rows, rng.choice((1, 4, 33)), page, heads=rng.choice((1, 3)), dim=rng.choice((64, 128)), seed=seed, scores=seed % 3 > 0,
             layout="token" if seed % 4 == 0 else "plain")
    for _ in range(14):
        parents = None if rng.random() < 0.3 else [b_ if rng.random() < 0.4 else rng.randrange(-2, rows + 2) for b_ in range(rows)]
        add = None if rng.random() < 0.1 else [rng.choice((0, 1, 1, rng.randrange(-3 * page, 4 * page))) for _ in range(rows)]
        b.update(parents, add)
        if rng.random() < 0.4:
            b.compact()


def test_large():
    """More rows than a wave has lanes, rows of many pages, pools that one look does not see whole."""
    b = Both(70003, 4096, 300, heads=1, seed=5, scores=False)
    rng = random.Random(3)
    b.update(None, [rng.randrange(0, 400) for _ in range(4096)])
    b.update([rng.randrange(-1, 4096) for _ in range(4096)], [rng.randrange(-50, 50) for _ in range(4096)])
    b.update([-1 if i % 3 else i for i in range(4096)], None)
    b.compact()
    b.update(None, [4800 if i == 1 else 16 * 300 + 1 if i == 4 else 1 for i in range(4096)])
    c = Both(70003, 3, 65536, heads=1, seed=6, scores=False)
    c.update(None, [65536 * 16, 5, 70000])          # all but a few pages
    c.update([1, 0, 1], [0, 1, 3])
    c.compact()
    c.update([-1, -1, 2], None)
    c.compact()


@pytest.mark.parametrize("pages", [4095, 4096, 4097, 20001, 32768, 32769, 36865])
def test_compaction_of_one_to_ten_blocks(pages):
    """Pools that every workgroup counts for itself, and those of a count beforehand; rows that are freed in front, between and at the end."""
    b = Both(pages, 5, pages, heads=1, seed=pages, scores=False)
    each = pages // 5
    for gone in ([0], [2, 4], [1, 2, 3]):
        b.update(None, [each * 16 - n for n in b.want.lens])
        b.update([-1 if i in gone else i for i in range(5)], [-16 * 77 if i == 3 else 0 for i in range(5)])
        b.compact()
    b.compact()


def test_edges():
    # the whole pool, to the last page, and one page too few
    b = Both(8, 3, 8)
    b.update(None, [5 * 16, 3 * 16, 1])
    b.update(None, [0, 0, 1])
    b.update(None, [-(5 * 16), 0, 1])
    b.update(None, [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1])
    b.update([5, -2 ** 31, 2 ** 31 - 1], [0, 0, 0])
    b.compact()   # of nothing
    # behind a row that finds too few none grows, not one that needs no page either
    b = Both(4, 3, 8)
    b.update(None, [17, 1, 0])
    b.update(None, [1, 1000, 1])
    b.update(None, [1, 100, 1])
    # a row at the end of the table: refused by itself, others go on
    b = Both(8, 2, 2)
    b.update(None, [32, 16])
    b.update(None, [1, 1])
    # forks that grow from within a page: each its own copy, also where all that share it write
    b = Both(12, 4, 3)
    b.update(None, [20, 0, 0, 0])
    b.update([0, 0, 0, 0], [1, 1, 0, 12])
    b.update([0, 0, 1, 2], [1, 1, 1, -10])
    b.update([3, 2, 1, 0], None)
    b.update([1, 0, 3, 2], [16, 1, 40, -3])


def test_counts_of_the_callers_own_and_pages_that_are_not_there():
    b = Both(10, 2, 4)
    b.update(None, [40, 0])
    keep = b.pool.page_table[0, :3].tolist()
    for x in keep:     # the prompt is kept
        b.want.refs[x] += 1
    b.pool.refs[torch.tensor(keep, device="cuda")] += 1
    b.update([-1, 0], [0, 1])      # written on from within: copied
    b.update([0, -1], [100, 0])    # never given out: too few
    b.compact()
    assert sum(b.want.refs) == 3
    b = Both(10, 2, 4)
    b.update(None, [60, 0])
    b.pool.page_table[0, 1] = b.want.table[0][1] = -1      # given away, by a caller that counts it out
    b.pool.page_table[0, 3] = b.want.table[0][3] = 77
    b.want.refs[1] = b.want.refs[3] = 0
    b.pool.refs[1] = b.pool.refs[3] = 0
    b.update([0, 0], [1, 2])       # from within a page that is not there: nothing to copy
    b.update([1, 0], [-15, 0])
    b.compact()


def test_the_same_as_torch_in_any_stream_and_captured():
    b = Both(40, 6, 5)
    parents, add, short = ints([0, 0, 0, 3, 3, 3]), ints([0, 5, 21, 0, 1, 30]), ints([9] * 6)
    b.update(None, [20, 0, 0, 37, 0, 0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    b.update([0, 0, 0, 3, 3, 3], [0, 5, 21, 0, 1, 30], stream=stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.update(b.k, b.v, parents, add, scores=b.scores, short=short)
        used = b.pool.compact(b.k, b.v, scores=b.scores)
    for steps in ([0, 1, 1, 0, 2, 2], [-1, 16, 3, 0, 0, 0], [4, 4, 4, -60, 9, 1], [0, 0, 0, 0, 0, 100]):
        add.copy_(ints(steps))
        graph.replay()
        want, copies = b.want.update([0, 0, 0, 3, 3, 3], steps)
        b.moved(copies)
        n, moves, _ = b.want.compact()
        b.moved(moves)
        b.check(steps)
        assert short.tolist() == want and used.tolist() == [n]


def test_layers_that_go_by_one_table():
    """Pairs of an update and of a compaction, for the caches of other layers and for all of them."""
    b = Both(40, 5, 6, heads=2)
    other = [(torch.randn_like(b.k), torch.randn_like(b.v)) for _ in range(2)]
    want = [(k.clone(), v.clone()) for k, v in other]
    copies, moves = torch.empty(5, 2, dtype=torch.int32, device="cuda"), torch.empty(40, 2, dtype=torch.int32, device="cuda")

    def follow(pairs):
        for k, v in other:
            paged.copy_pages(k, v, k, v, pairs)
        made = [p for p in pairs.tolist() if p != [-1, -1]]
        for k, v in want:
            for x in (k, v):
                if made:
                    s, t = (torch.tensor(y, device="cuda") for y in zip(*made))
                    x[t] = x[s]
        assert all(torch.equal(x, y) for a, c in zip(other, want) for x, y in zip(a, c))
        return made

    b.update(None, [20, 33, 0, 7, 0])
    for parents, add in (([0, 0, 1, 0, 1], [1, 2, 3, 0, -4]), ([0, 1, 4, 4, 4], [5, 0, 1, 1, 1]), ([0, 1, -1, 2, 3], [0, 0, 90, 0, 0])):
        _, pairs = b.want.update(parents, add)
        b.moved(pairs)
        b.pool.update(b.k, b.v, ints(parents), ints(add), scores=b.scores, copies=copies)
        b.check(parents)
        assert [tuple(p) for p in follow(copies)] == pairs
        before = [x.clone() for x in (b.k, b.v)]
        n, pairs, _ = b.want.compact()
        assert b.pool.compact(None, None, moves=moves).tolist() == [n]    # this layer too by the pairs
        assert torch.equal(b.k, before[0]) and torch.equal(b.v, before[1])
        assert [tuple(p) for p in follow(moves)] == pairs
        paged.copy_pages(b.k, b.v, b.k, b.v, moves, b.scores, b.scores)
        b.moved(pairs)
        b.check("compact")
    b.want.update([0, 0, 0, 0, 0], [1, 1, 1, 1, 1])
    short = b.pool.update(None, None, ints([0, 0, 0, 0, 0]), ints([1, 1, 1, 1, 1]), copies=copies)
    assert b.pool.page_table.tolist() == b.want.table and not short.any()
    for call in (lambda: b.pool.update(None, None), lambda: b.pool.compact(None, None), lambda: b.pool.update(None, b.v, copies=copies),
                 lambda: b.pool.update(None, None, copies=copies[:4]), lambda: b.pool.update(b.k, b.v, copies=copies.float())):
        with pytest.raises(ValueError):
            call()


def test_offsets_past_32_bits():
    """Pages behind the first 2^32 elements: forks that are copied there and back, compaction to the front."""
    pages = 2 ** 22 + 6    # of 16 x 64, one head
    k, v = (torch.zeros(pages, 1, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    scores = torch.zeros(pages, 1, 16, device="cuda")
    pool = paged.PagePool(pages, 2, 4, 16)
    pool.refs[:-4] = 1    # of the caller's own
    pool.update(k, v, add=ints([20, 0]), scores=scores)
    assert pool.page_table.tolist()[0] == [pages - 4, pages - 3, -1, -1]
    g = torch.Generator(device="cuda").manual_seed(1)
    for x in (k, v, scores):
        x[-4:-2].copy_(torch.randn(x[-4:-2].shape, generator=g, device="cuda"))
    kept = [x[-4:-2].clone() for x in (k, v, scores)]
    pool.update(k, v, ints([0, 0]), ints([0, 3]), scores=scores)
    assert pool.page_table.tolist()[1] == [pages - 4, pages - 2, -1, -1] and pool.refs[-4:].tolist() == [2, 1, 1, 0]
    for x, want in zip((k, v, scores), kept):
        assert torch.equal(x[-2], want[1]) and not x[-1].any()
    pool.refs[5:-4] = 0
    assert pool.compact(k, v, scores=scores).tolist() == [8] and pool.page_table.tolist() == [[5, 6, -1, -1], [5, 7, -1, -1]]
    for x, want in zip((k, v, scores), kept):
        assert torch.equal(x[5:7], want) and torch.equal(x[7], want[1])


def test_copy_pages():
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(9, 3, 32, 128, generator=g, device="cuda").half() for _ in range(2))
    s = torch.randn(9, 3, 32, generator=g, device="cuda")
    to = [torch.zeros(6, 32, 3, 136, dtype=torch.float16, device="cuda")[..., :128].permute(0, 2, 1, 3) for _ in range(2)]
    st = torch.zeros(6, 3, 32, device="cuda")
    pairs = [(0, 5), (8, 0), (0, 3), (-1, 1), (9, 1), (4, 6), (4, -1)]
    paged.copy_pages(k, v, *to, ints(pairs), s, st)
    for x, y in ((k, to[0]), (v, to[1]), (s, st)):
        want = torch.zeros_like(y)
        for a, b in pairs[:3]:
            want[b] = x[a]
        assert torch.equal(y, want)
    before = k.clone()
    paged.copy_pages(k, v, k, v, ints([(1, 2), (1, 7)]))
    assert torch.equal(k[2], before[1]) and torch.equal(k[7], before[1]) and torch.equal(k[[0, 1, 3, 4, 5, 6, 8]], before[[0, 1, 3, 4, 5, 6, 8]])
    paged.copy_pages(k, v, k, v, torch.zeros(0, 2, dtype=torch.int32, device="cuda"))


def test_refusals():
    b = Both(10, 2, 4)
    k, v, pool = b.k, b.v, b.pool
    for call in (lambda: pool.update(k[:9], v[:9]), lambda: pool.update(k, v[:, :, :, :32]), lambda: pool.update(k, v, ints([0])), lambda: pool.update(k, v, add=torch.zeros(2, device="cuda")),
                 lambda: pool.update(k, v, ints([0, 1]).cpu()), lambda: pool.update(k, v, short=ints([0] * 3)), lambda: pool.update(k, v.half()), lambda: pool.update(k, v, scores=b.scores[:, :1]),
                 lambda: pool.compact(k, v, used=ints([0, 0])), lambda: pool.compact(k, v, moved=ints([0])), lambda: paged.copy_pages(k, v, k.half(), v.half(), ints([[0, 1]])),
                 lambda: paged.copy_pages(k, v, k, v, ints([0, 1])), lambda: paged.copy_pages(k, v, k, v, ints([[0, 1]]), b.scores)):
        with pytest.raises(ValueError):
            call()
    b.check("nothing has changed")


def test_a_serving_loop():
    """Prompts, forks and single tokens by way of everything: pages from the pool, rotary positions on the way into the cache, capped attention, a
    compaction in between -- against one long sequence for every row, attended as a whole."""
    from ringattention_amd.rotary import Rotary
    H, HKV, D, page = 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = paged.PagePool(64, 4, 8, page)
    k_cache, v_cache = (torch.zeros(64, HKV, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    plan = paged.PagedAttention(H, D, kv_heads=HKV, dtype="fp16", page_size=page, max_batch=4, max_tokens=128, softcap=15.0)
    rotary = Rotary(D, 32, interleaved=True, scaling="ntk", factor=4, dtype="fp16")
    rows = {b: [] for b in range(4)}    # what every row's sequence is made of: (q, k, v) of its tokens

    def step(parents, add):
        short = pool.update(k_cache, v_cache, ints(parents), ints(add))
        assert not short.any()
        n = sum(add)
        q, k, v = (torch.randn(n, h, D, generator=g, device="cuda").half() for h in (H, HKV, HKV))
        starts = ints([sum(add[:b]) for b in range(5)])
        seqs = (pool.page_table, pool.lens, starts)
        turned = plan.append_rotary(rotary, q, k, v, k_cache, v_cache, *seqs)
        out, lse = plan.forward(turned, k_cache, v_cache, *seqs)
        old = dict(rows)
        for b in range(4):
            at = sum(add[:b])
            rows[b] = (list(old[parents[b]]) if parents[b] >= 0 else []) + [(q[at + i], k[at + i], v[at + i]) for i in range(add[b])]
        for b in range(4):
            assert len(rows[b]) == int(pool.lens[b])
            if not add[b]:
                continue
            Q, K, V = (torch.stack(x) for x in zip(*rows[b]))
            Q, K = rotary.apply(Q, K)
            group = H // HKV
            Q, K, V = Q.double(), K.double().repeat_interleave(group, 1), V.double().repeat_interleave(group, 1)
            x = torch.einsum("ihd,jhd->hij", Q.cpu(), K.cpu()) / D ** 0.5
            x = 15 * torch.tanh(x / 15)
            x = x.masked_fill(torch.ones(x.shape[1:], dtype=torch.bool).triu(1), float("-inf"))
            p = torch.softmax(x, dim=-1)
            o = torch.einsum("hij,jhd->ihd", p, V.cpu())
            size = torch.einsum("hij,jhd->ihd", p, V.cpu().abs())
            n, at = add[b], sum(add[:b])
            # probabilities and O in fp16 (half a step each), scores in 32 bits
            tol = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -13) * size + 2.0 ** -20
            assert ((out[at:at + n].double().cpu() - o[-n:]).abs() <= tol[-n:]).all(), b

    step([-1, -1, -1, -1], [37, 20, 0, 0])
    step([0, 1, 0, 0], [1, 1, 1, 1])        # two forks of the first, all write on
    step([0, 1, 2, 2], [1, 16, 1, 3])
    pool.compact(k_cache, v_cache)
    step([2, -1, 2, 3], [1, 30, 0, 1])      # one ends, a new prompt in its place; another becomes a fork
    pool.compact(k_cache, v_cache)
    step([0, 1, 2, 1], [2, 1, 5, 9])
