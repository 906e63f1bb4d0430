"""Serving from a paged K/V cache, as cases that can be timed: the cache's append, attention of new tokens over it (causal, and
with a sliding window beside a few first tokens that stay visible), the attention weight that every cached token has drawn, and the
eviction that keeps the tokens that drew most.

    listed()          the cases by name
    draw(rng)         one more case of the same ranges
    prepare(case, s)  what a program holds before the call: the pool of pages, tables, lengths, new tokens, and the plan
    run(state)        one pass through an operator, and its outputs
    work(case)        bytes and operations a pass cannot do without
    exact(case, s)    what run() returns, from the definition in 64 bits

A case is a dict of plain values:
    op      "append", "attend", "weights" or "evict"
    lens    tokens of every sequence in the cache, the new ones among them, "1024*64" or "640,512,384"
    news    new tokens of every sequence, its last ones ("evict": none)
    heads, kv_heads, dim, dtype, page (tokens of a page)
    window, sinks   a query sees the last `window` tokens up to itself and the first `sinks` (0, 0: all up to itself)
    head_major      the new tokens' tensors lie head by head in memory instead of token by token
    budget, first, last   evict: tokens kept of a sequence; the first and the last ones stay whatever they drew

A pool is [pages, kv_heads, page, dim]; a sequence's pages lie in it in no order.  With `own` run() calls the package, else elementary torch.
"""
import math

import torch

own = False

TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEFAULTS = {"heads": 8, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "window": 0, "sinks": 0, "head_major": False, "budget": 0, "first": 0, "last": 0}


def _case(op, lens, news="", **more):
    return dict(DEFAULTS, op=op, lens=lens, news=news, **more)


def listed():
    return [
        # a step of a serving loop: one token of each of 64 sequences goes into the cache
        _case("append", "1024*64", "1*64", name="append_step"),
        # prompts of uneven length go in at once, 8 K tokens of a 32-head model
        _case("append", "1021,777,1300,64,905,333,2048,1744", "1021,777,1300,64,905,333,2048,1744", name="append_prompts", heads=32, kv_heads=32, page=16),
        # the smallest call: one token over 512, eight heads of 64, fp16; what counts is the launch and the latency of a short walk
        _case("attend", "512", "1", name="token_short", dim=64, dtype="fp16"),
        # a serving step: a token of each of 48 sequences of uneven length, grouped heads
        _case("attend", ",".join(str(128 + (i * 2659) % 7919) for i in range(48)), "1*48", name="tokens_batch", heads=16, kv_heads=4),
        # one token of one sequence of 128 K tokens: few rows, a long walk
        _case("attend", "131072", "1", name="token_long", heads=16, kv_heads=16, dtype="fp16", page=256),
        # the next 4096 tokens of a prompt of 32 K, 32 heads: a chunk of a long prefill
        _case("attend", "32768", "4096", name="chunk_32k", heads=32, kv_heads=32),
        # a batch of a prompt's chunk next to sequences that take a token or a few each, ragged, small pages, head-major tensors
        _case("attend", "2309,905,4096,333,1300,5000,64,777,3001,1", "509,1,1,7,1,2,64,1,1,1", name="mixed_batch", heads=16, kv_heads=4, page=16, head_major=True),
        # the same chunk of a model with a sliding window of 1024 and four first tokens that stay
        _case("attend", "32768", "4096", name="chunk_window", heads=32, kv_heads=8, window=1024, sinks=4),
        # the weights that a serving step's tokens give to the cached ones
        _case("weights", ",".join(str(128 + (i * 2659) % 7919) for i in range(48)), "1*48", name="weights_step", heads=16, kv_heads=4),
        # the weights within a prompt of 8 K tokens
        _case("weights", "8192", "8192", name="weights_prompt", heads=16, kv_heads=4, dtype="fp16"),
        # sixteen sequences of some 8 K tokens shrink to 4096 each
        _case("evict", ",".join(str(7168 + (i * 541) % 1021) for i in range(16)), name="evict_batch", heads=8, kv_heads=8, budget=4096, first=4, last=256),
        # one sequence of 128 K tokens keeps a quarter
        _case("evict", "131072", name="evict_long", heads=16, kv_heads=4, dtype="fp16", page=256, budget=32768, first=4, last=1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


MAX_FLOPS = 1.5e12      # a drawn case does at most this (the largest listed one does 2.1e12)
MAX_SCORES = 2.5e9      # padded scores of a drawn case's plain form (the largest listed one has 4.3e9)
MAX_CACHE = 2 ** 31     # bytes of K and V of a drawn case


def draw(rng):
    """1 to 128 sequences of 1 to 100 K tokens, chunks of 1 to 4096 new tokens, 1 to 32 heads in groups of 1 to 8, pages of 16 to 256."""
    while True:
        op = rng.choice(("append", "attend", "attend", "attend", "attend", "weights", "weights", "evict", "evict"))
        group = rng.choice((1, 1, 2, 4, 8))
        kv = rng.choice((1, 2, 4, 8, 16, 32))
        if group * kv > 32:
            continue
        batch = _log_int(rng, 1, 128)
        longest = _log_int(rng, 1 if op != "evict" else 64, 100000)
        lens = [longest] + [max(1, int(longest * rng.random())) for _ in range(batch - 1)]
        c = _case(op, "", heads=group * kv, kv_heads=kv, dim=rng.choice((64, 128)), dtype=rng.choice(("fp16", "bf16")), page=rng.choice((16, 32, 64, 128, 256)))
        if op == "evict":
            c["budget"] = max(1, int(longest * (0.1 + 0.8 * rng.random())))
            c["first"] = min(rng.choice((0, 1, 4)), c["budget"])
            c["last"] = int((c["budget"] - c["first"]) * 0.3 * rng.random())
        else:
            kind = rng.choice(("token", "chunk", "mixed"))
            most = _log_int(rng, 2, 4096)
            news = [1 if kind == "token" or (kind == "mixed" and rng.random() < 0.7) else max(1, min(n, int(most * (0.3 + 0.7 * rng.random())))) for n in lens]
            if kind == "mixed" and batch > 2:
                news[rng.randrange(1, batch)] = 0   # a sequence that has nothing new in this call
            c["news"] = ",".join(map(str, news))
            c["head_major"] = rng.random() < 0.3
            if op in ("attend", "weights") and rng.random() < 0.4:
                c["window"] = _log_int(rng, 16, 8192)
                c["sinks"] = rng.choice((0, 1, 4, 64))
        c["lens"] = ",".join(map(str, lens))
        if sum(lens) * kv * c["dim"] * 4 > MAX_CACHE:
            continue
        if op in ("attend", "weights") and (work(c)["flops"] > MAX_FLOPS or batch * max(_ints(c["news"])) * c["heads"] * longest > MAX_SCORES):
            continue
        return c


def _ints(text):
    if "*" in text:
        n, times = text.split("*")
        return [int(n)] * int(times)
    return [int(x) for x in text.split(",")] if text else []


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, hkv, d = TORCH[c["dtype"]], c["page"], c["kv_heads"], c["dim"]
    lens, news = _ints(c["lens"]), _ints(c["news"])

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    def table(needed, first):
        """The pages of every sequence, in no order; -1 behind its last."""
        order = (torch.randperm(sum(needed), generator=gen, device="cuda", dtype=torch.int64) + first).to(torch.int32)
        t = torch.full((len(needed), max(needed)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(needed):
            t[b, :n] = order[at:at + n]
            at += n
        return t

    pages = [-(-n // page) for n in lens]
    total = sum(pages)
    s = {"case": c, "table": table(pages, 0), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    if c["op"] == "evict":
        s["kept_table"] = table([-(-c["budget"] // page)] * len(lens), total)
        total += s["kept_table"].numel()
    s["k_cache"], s["v_cache"] = normal(total, hkv, page, d), normal(total, hkv, page, d)
    if c["op"] in ("weights", "evict"):
        # weights drawn so far: a few tokens draw most, many next to nothing or nothing at all
        x = torch.randn((total, hkv, page), generator=gen, device="cuda")
        s["scores"] = torch.relu(torch.exp(2 * x) - 0.05)
    if c["op"] != "evict":
        T = sum(news)
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        heads = c["heads"] if c["op"] in ("attend", "weights") else hkv

        def new_tokens(h):
            return normal(h, T, d).transpose(0, 1) if c["head_major"] else normal(T, h, d)

        if c["op"] == "append":
            s["k"], s["v"] = new_tokens(heads), new_tokens(heads)
        else:
            s["q"] = new_tokens(heads)
        if c["op"] == "weights":
            s["lse"] = _plain_attend(s)[1]
    if own:
        from ringattention_amd import paged
        s["plan"] = paged.PagedAttention(c["heads"], d, kv_heads=hkv, dtype=c["dtype"], page_size=page, max_batch=len(lens),
                                         max_tokens=max(1, sum(news)), window=c["window"], sinks=c["sinks"])
        if c["op"] == "attend":
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(c["heads"], s["q"].shape[0], dtype=torch.float32, device="cuda")
        if c["op"] == "evict":
            s["kept"] = torch.empty(len(lens), hkv, c["budget"], dtype=torch.int32, device="cuda")
            s["kept_lens"] = torch.empty(len(lens), dtype=torch.int32, device="cuda")
    return s


def _token_places(s):
    """Of every new token: its sequence, its number among that one's new tokens, its position in the sequence."""
    starts = s["starts"].long()
    t = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(starts, t, right=True) - 1
    i = t - starts[b]
    return b, i, s["lens"].long()[b] - (starts[b + 1] - starts[b]) + i


def _padded_scores(s):
    """(scaled scores [batch, kv_heads, new tokens x heads of a group, keys] in 32 bits with -inf where a key is hidden, sequence and number of every token)"""
    c = s["case"]
    hkv, group, d, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["page"]
    s = dict(s, T=s["q"].shape[0])
    b, i, _ = _token_places(s)
    most = max(_ints(c["news"]))
    starts, lens = s["starts"].long(), s["lens"].long()
    n = starts[1:] - starts[:-1]
    at = torch.arange(most, device="cuda")
    tokens = (starts[:-1, None] + torch.minimum(at[None, :], (n - 1).clamp(min=0)[:, None])).clamp(max=s["T"] - 1)
    q = s["q"][tokens].float().reshape(len(lens), most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(len(lens), hkv, most * group, d)
    k = _gathered(s["k_cache"], s["table"])
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(d))
    del k
    key = torch.arange(scores.shape[3], device="cuda")
    place = (lens - n)[:, None] + at[None, :]
    seen = (key <= place[:, :, None]) & (key < lens[:, None, None]) & (at[None, :] < n[:, None])[:, :, None]
    if c["window"]:
        seen &= (key > place[:, :, None] - c["window"]) | (key < c["sinks"])
    seen = seen.repeat_interleave(group, dim=1)[:, None]
    return scores.masked_fill_(~seen, -math.inf), b, i


def _gathered(cache, table):
    """The sequences' rows of a cache in 32 bits, [batch, kv_heads, keys, dim]."""
    x = cache[table.long().clamp(min=0)].float()
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _plain_attend(s):
    c = s["case"]
    hkv, group, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    scores, b, i = _padded_scores(s)
    top = scores.amax(dim=3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(dim=3, keepdim=True)
    o = torch.matmul(p, _gathered(s["v_cache"], s["table"])) / torch.where(total == 0, 1.0, total)
    lse = (total.log() + top)[..., 0]
    most = o.shape[2] // group
    o = o.reshape(-1, hkv, most, group, d)[b, :, i].reshape(-1, c["heads"], d)   # [tokens, heads, dim]
    lse = lse.reshape(-1, hkv, most, group)[b, :, i].reshape(-1, c["heads"])
    return o.to(s["q"].dtype), lse.transpose(0, 1).contiguous()


def _plain_weights(s):
    c = s["case"]
    hkv, group, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    scores, b, i = _padded_scores(s)
    most = scores.shape[2] // group
    # the LSE of every padded row: those without a token have no visible key
    lse = torch.zeros(scores.shape[:3], device="cuda").reshape(-1, hkv, most, group)
    lse[b, :, i] = s["lse"].transpose(0, 1).reshape(-1, hkv, group)
    w = scores.sub_(lse.reshape(scores.shape[:3])[..., None]).exp_().sum(dim=2)   # [batch, kv_heads, keys]
    table = s["table"].long().clamp(min=0)
    at = (table[:, None, :, None] * hkv + torch.arange(hkv, device="cuda")[None, :, None, None]) * page + torch.arange(page, device="cuda")
    s["scores"].view(-1).scatter_add_(0, at.reshape(-1), w.reshape(-1))
    return s["scores"]


def _plain_evict(s):
    c = s["case"]
    page, budget = c["page"], c["budget"]
    table, lens, to = s["table"].long().clamp(min=0), s["lens"].long(), s["kept_table"].long()
    x = s["scores"][table].permute(0, 2, 1, 3)
    x = x.reshape(x.shape[0], x.shape[1], -1)
    key = torch.arange(x.shape[2], device="cuda")
    n = lens[:, None, None]
    stays = (key < c["first"]) | (key >= n - c["last"])
    rank = torch.where(stays, math.inf, torch.where(torch.isnan(x), -math.inf, x).double())
    # places behind a sequence's end come after everything else
    order = torch.where(key < n, rank, -math.inf).sort(dim=2, descending=True, stable=True).indices
    order = torch.where(order < n, order, x.shape[2])
    picked = order[:, :, :budget].sort(dim=2).values
    kept_lens = torch.clamp(lens, max=budget)
    there = torch.arange(budget, device="cuda") < kept_lens[:, None, None]
    b = torch.arange(len(lens), device="cuda")[:, None, None]
    h = torch.arange(c["kv_heads"], device="cuda")[None, :, None]
    at = picked.clamp(max=x.shape[2] - 1)
    j = torch.arange(budget, device="cuda")
    src = (table[b, at // page], h, at % page)
    dst = (to[b, j // page], h, j % page)
    for_rows = there[..., None]
    s["k_cache"][dst] = torch.where(for_rows, s["k_cache"][src], s["k_cache"][dst])
    s["v_cache"][dst] = torch.where(for_rows, s["v_cache"][src], s["v_cache"][dst])
    s["scores"][dst] = torch.where(there, s["scores"][src], s["scores"][dst])
    kept = torch.where(there, picked, -1).to(torch.int32)
    return s["k_cache"], s["v_cache"], s["scores"], kept, kept_lens.to(torch.int32)


def _plain_append(s):
    page = s["case"]["page"]
    b, _, place = _token_places(dict(s, T=s["k"].shape[0]))
    pages = s["table"].long()[b, place // page]
    s["k_cache"][pages, :, place % page] = s["k"]
    s["v_cache"][pages, :, place % page] = s["v"]
    return s["k_cache"], s["v_cache"]


def run(s):
    c = s["case"]
    if own:
        plan, cache = s["plan"], (s["k_cache"], s["v_cache"])
        if c["op"] == "append":
            plan.append(s["k"], s["v"], *cache, s["table"], s["lens"], s["starts"])
            return cache
        if c["op"] == "attend":
            return plan.forward(s["q"], *cache, s["table"], s["lens"], s["starts"], s["out"], s["lse"])
        if c["op"] == "weights":
            return plan.weights(s["q"], s["lse"], s["k_cache"], s["table"], s["lens"], s["starts"], s["scores"])
        kept, kept_lens = plan.evict(*cache, s["scores"], s["table"], s["lens"], s["kept_table"], c["budget"], c["first"], c["last"], s["kept"], s["kept_lens"])
        return cache + (s["scores"], kept, kept_lens)
    if c["op"] == "append":
        return _plain_append(s)
    if c["op"] == "attend":
        return _plain_attend(s)
    return _plain_weights(s) if c["op"] == "weights" else _plain_evict(s)


def _pairs(length, new, window, sinks):
    """Visible (query, key) pairs of a head of a sequence, and its keys that some query sees."""
    first = length - new
    if not window:
        return new * first + new * (new + 1) // 2, length if new else 0
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(first, length))
    low = max(0, first + 1 - window)
    return pairs, length - low + min(sinks, low) if new else 0


def work(case):
    c = case
    lens, news = _ints(c["lens"]), _ints(c["news"])
    hkv, H, d = c["kv_heads"], c["heads"], c["dim"]
    if c["op"] == "append":   # the new rows of K and V, read and written
        return {"bytes": sum(news) * hkv * d * 2 * 4, "flops": 0}
    if c["op"] == "evict":   # every score once; of a kept token K, V and score, read and written, and its number
        kept = sum(min(n, c["budget"]) for n in lens)
        return {"bytes": hkv * (sum(lens) * 4 + kept * (8 * d + 8)), "flops": 0}
    both = [_pairs(n, m, c["window"], c["sinks"]) for n, m in zip(lens, news)]
    pairs, keys = sum(x[0] for x in both), sum(x[1] for x in both)
    if c["op"] == "attend":   # K and V that are seen, Q and O, LSE
        return {"bytes": keys * hkv * d * 4 + sum(news) * H * (4 * d + 4), "flops": 4 * d * H * pairs}
    # weights: K, Q and LSE; a score of every key read and written
    return {"bytes": keys * hkv * (2 * d + 8) + sum(news) * H * (2 * d + 4), "flops": 2 * d * H * pairs}


def exact(case, seed):
    """Sequence by sequence and head by head in 64 bits: rows of a cache by (page, slot), sums over what a query sees."""
    c = case
    if c["op"] in ("append", "evict"):
        return None   # rows are copied, none computed
    s = prepare(case, seed)
    lens, news, page = _ints(c["lens"]), _ints(c["news"]), c["page"]
    hkv, group, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]

    def rows(cache, b, h, n):
        pages = s["table"][b, :-(-n // page)].long()
        return cache[pages, h].reshape(-1, *cache.shape[3:])[:n]

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(c["heads"], s["q"].shape[0], dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if c["op"] == "weights" else None
    for b, (n, m) in enumerate(zip(lens, news)):
        at = int(s["starts"][b])
        for h in range(hkv if m else 0):
            k = rows(s["k_cache"], b, h, n).double()
            v = rows(s["v_cache"], b, h, n).double() if c["op"] == "attend" else None
            drawn = torch.zeros(n, dtype=torch.float64, device="cuda")
            for i in range(0, m, 512):
                some = range(i, min(m, i + 512))
                place = torch.tensor([n - m + x for x in some], device="cuda")[:, None]
                key = torch.arange(n, device="cuda")[None, :]
                hidden = key > place
                if c["window"]:
                    hidden |= (place - key >= c["window"]) & (key >= c["sinks"])
                for g in range(h * group, (h + 1) * group):
                    x = s["q"][at + i:at + i + len(some), g].double() @ k.t() / d ** 0.5
                    x = x.masked_fill(hidden, -math.inf)
                    if c["op"] == "attend":
                        z = torch.logsumexp(x, dim=1)
                        lse[g, at + i:at + i + len(some)] = z
                        out[at + i:at + i + len(some), g] = torch.exp(x - z[:, None]) @ v
                    else:
                        drawn += torch.exp(x - s["lse"][g, at + i:at + i + len(some)].double()[:, None]).sum(dim=0)
            if scores is not None:
                key = torch.arange(n, device="cuda")
                scores[s["table"][b].long()[key // page], h, key % page] += drawn
    return (out, lse) if c["op"] == "attend" else scores
