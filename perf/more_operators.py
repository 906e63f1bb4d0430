"""What a served model puts around a paged K/V cache, as cases that can be timed: rotary positions, attention whose scores are capped,
biased by distance or masked by documents and prefixes, and the pages' bookkeeping -- forks, growth, compaction.

    listed()          the cases by name
    draw(rng)         one more case of the same ranges
    prepare(case, s)  what a program holds before the call: tensors, tables, lengths, frequencies, and the plan
    run(state)        one pass through an operator, and its outputs
    work(case)        bytes and operations a pass cannot do without
    exact(case, s)    what run() returns, from the definition in 64 bits

A case is a dict of plain values:
    op      "rotate"   rotary positions of Q and K of a sequence [batch, heads, tokens, dim] (a ring's tensors)
            "append"   rotary positions of a call's new tokens: Q turned, K turned and V as they are into the cache
            "attend"   attention of new tokens over the cache with a cap, slopes, prefixes or documents
            "weights"  the attention weight that cached tokens drew in such a call
            "fork"     rows of the page table become forks of others or begin anew, and grow: counts, table, copied pages
            "compact"  the pages in use move to the front of the pool
    lens    tokens of every sequence in the cache, the new ones among them, "1024*64" or "640,512,384"
    news    new tokens of every sequence, its last ones
    heads, kv_heads, dim, dtype, page (tokens of a page)
    tokens, ranks   rotate: length of the sequence; 0 or how many ranks' low and high halves its rows lie in (zigzag)
    turned, interleaved, inverse, scaling, spread   rotary: columns that turn, how they pair up, back instead of forth, "" or "linear" or
            "ntk" or "yarn", and how many times longer than trained
    cap, slopes, prefix, docs, window, sinks   scores: cap of their tanh; a slope for every head; tokens at the beginning that every token sees;
            tokens of a document (0: one document); sliding window and first tokens that stay visible
    groups, spare   fork: rows that share a parent, itself among them; compact: every so-many-th page is in use

A pool is [pages, kv_heads, page, dim]; a sequence's pages lie in it in no order.  With `own` run() calls the package, else elementary torch.
"""
import math

import torch

own = False

TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEFAULTS = {"heads": 8, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "lens": "", "news": ""}
ROTARY = {"turned": 128, "interleaved": False, "inverse": False, "scaling": "", "spread": 1}
SCORES = {"cap": 0.0, "slopes": False, "prefix": 0, "docs": 0, "window": 0, "sinks": 0}
BASE = 10000.0
TRAINED = 4096    # tokens that "yarn" takes the model to have been trained on
STEP = ",".join(str(128 + (i * 2659) % 7919) for i in range(48))   # 48 sequences of uneven length


def _case(op, **more):
    kind = ROTARY if op in ("rotate", "append") else SCORES if op in ("attend", "weights") else {}
    return {**DEFAULTS, **kind, "op": op, **more}


def listed():
    return [
        # a long context's Q and K before the ring: 32 K tokens, grouped heads, zigzag placement over 8 ranks, frequencies stretched by 8
        _case("rotate", name="rotate_ring", tokens=32768, ranks=8, heads=32, kv_heads=8, scaling="yarn", spread=8),
        # gradients of a shorter odd one turned back: interleaved pairs, half of a row of 128, fp16
        _case("rotate", name="rotate_back", tokens=4093, ranks=0, heads=16, kv_heads=4, turned=64, interleaved=True, inverse=True, dtype="fp16"),
        # a step of a serving loop: one token of each of 48 sequences; what counts is the launch
        _case("append", name="append_step", lens=STEP, news="1*48", heads=32, kv_heads=8, scaling="linear", spread=4),
        # prompts of uneven length, 8 K tokens at once, small pages
        _case("append", name="append_prompts", lens="1021,777,1300,64,905,333,2048,1744", news="1021,777,1300,64,905,333,2048,1744", heads=32, kv_heads=32, page=16),
        # the smallest attention: a token over 512 with capped scores
        _case("attend", name="cap_token", lens="512", news="1", dim=64, dtype="fp16", cap=50.0),
        # a serving step with capped scores, grouped heads
        _case("attend", name="cap_step", lens=STEP, news="1*48", heads=16, kv_heads=4, cap=50.0),
        # the next 4096 tokens of a prompt of 32 K with capped scores
        _case("attend", name="cap_chunk", lens="32768", news="4096", heads=32, kv_heads=8, cap=50.0),
        # a ragged batch of prompts' chunks and single tokens under slopes, with prefixes that all tokens see
        _case("attend", name="slope_mixed", lens="4099,905,4096,333,1300,5000,64,777", news="4099,1,1024,7,1300,2,64,1", heads=16, kv_heads=16, dtype="fp16", slopes=True, prefix=100, page=16),
        # documents packed one behind the other into a sequence of 16 K
        _case("attend", name="documents", lens="16384", news="16384", heads=16, kv_heads=4, docs=1365),
        # the weights within a prompt of 8 K with capped scores and slopes
        _case("weights", name="weights_prompt", lens="8192", news="8192", heads=16, kv_heads=4, dtype="fp16", cap=30.0, slopes=True),
        # beams: 16 prompts with 8 rows each, 7 of which become forks of the first and take a token more
        _case("fork", name="fork_beams", lens="2049*128", groups=8, kv_heads=8),
        # a pool of which two pages in five are in use
        _case("compact", name="compact_pool", lens="3001*24", spare=5, kv_heads=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


MAX_FLOPS = 6e11        # a drawn case does at most this (the largest listed one does 2e12)
MAX_SCORES = 3e9        # scores of a drawn case's plain form, padded
MAX_BYTES = 2 ** 31     # K and V of a drawn case's pool, or Q and K of a ring


def draw(rng):
    """1 to 128 sequences of 1 to 64 K tokens, chunks of 1 to 4096 new tokens, 1 to 32 heads in groups of 1 to 8, pages of 16 to 256."""
    while True:
        op = rng.choice(("rotate", "append", "append", "attend", "attend", "attend", "weights", "fork", "compact"))
        group, kv = rng.choice((1, 1, 2, 4, 8)), rng.choice((1, 2, 4, 8, 16, 32))
        if group * kv > 32:
            continue
        c = _case(op, heads=group * kv, kv_heads=kv)
        c.update(dim=rng.choice((64, 128)), dtype=rng.choice(("fp16", "bf16")), page=rng.choice((16, 32, 64, 128, 256)))
        if op in ("rotate", "append"):
            c.update(turned=rng.choice((16, 32, 48, c["dim"], c["dim"], c["dim"])), interleaved=rng.random() < 0.4, scaling=rng.choice(("", "linear", "ntk", "yarn")))
            c["spread"] = rng.choice((2, 4, 8, 32)) if c["scaling"] else 1
        if op == "rotate":
            c.update(inverse=rng.random() < 0.5, ranks=rng.choice((0, 0, 2, 4, 8)))
            c["tokens"] = _log_int(rng, 1, 65536)
            if c["ranks"]:
                c["tokens"] = -(-c["tokens"] // (2 * c["ranks"])) * 2 * c["ranks"]
            if c["tokens"] * (group + 1) * kv * c["dim"] * 2 <= MAX_BYTES:
                return c
            continue
        batch, longest = _log_int(rng, 1, 128), _log_int(rng, 1, 65536)
        lens = [longest] + [max(1, int(longest * rng.random())) for _ in range(batch - 1)]
        if op == "fork":
            c["groups"] = rng.choice((2, 3, 4, 8, 16))
            lens = [lens[i // c["groups"]] for i in range(batch)]
        if op == "compact":
            c["spare"] = rng.choice((2, 3, 5, 9))
        c["lens"] = ",".join(map(str, lens))
        if sum(-(-n // c["page"]) + 1 for n in lens) * c["page"] * kv * c["dim"] * 4 * c.get("spare", 1) > MAX_BYTES:
            continue
        if op in ("fork", "compact"):
            return c
        kind, most = rng.choice(("token", "chunk", "mixed")), _log_int(rng, 2, 4096)
        news = [1 if kind == "token" or (kind == "mixed" and rng.random() < 0.7) else max(1, min(n, int(most * (0.3 + 0.7 * rng.random())))) for n in lens]
        if kind == "mixed" and batch > 2:
            news[rng.randrange(1, batch)] = 0   # a sequence that has nothing new in this call
        c["news"] = ",".join(map(str, news))
        if op in ("attend", "weights"):
            c["cap"] = rng.choice((0.0, 20.0, 30.0, 50.0))
            c["slopes"] = rng.random() < 0.4
            if rng.random() < 0.3:
                c.update(window=_log_int(rng, 16, 8192), sinks=rng.choice((0, 1, 4, 64)))
            if rng.random() < 0.3:
                c["prefix"] = _log_int(rng, 1, 2048)
            if rng.random() < 0.3 or not (c["cap"] or c["slopes"] or c["prefix"]):
                c["docs"] = _log_int(rng, 3, 4096)
            if _pairs_bound(lens, news) * c["heads"] * 4 * c["dim"] > MAX_FLOPS or batch * max(news) * c["heads"] * longest > MAX_SCORES:
                continue
        return c


def _ints(text):
    if "*" in text:
        n, times = text.split("*")
        return [int(n)] * int(times)
    return [int(x) for x in text.split(",")] if text else []


def _pairs_bound(lens, news):
    return sum(n * m for n, m in zip(lens, news))


# ---- the definitions' numbers: frequencies, slopes, documents, placement

def _frequencies(c):
    """(radians per position of every pair, in 64 bits; what turned columns are multiplied by)"""
    half, s = c["turned"] // 2, float(c["spread"])
    base = BASE * s ** (2 * half / (2 * half - 2)) if c["scaling"] == "ntk" and half > 1 else BASE
    f = [base ** (-i / half) for i in range(half)]
    if c["scaling"] == "linear":
        f = [x / s for x in f]
    if c["scaling"] == "yarn":   # pairs that turn more than 32 times within what was trained stay, those that turn less than once are stretched
        def pair(turns):
            return half * math.log(TRAINED / (turns * 2 * math.pi)) / math.log(BASE)
        low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), 2 * half - 1)
        stays = [1 - min(max((i - low) / max(high - low, 0.001), 0), 1) for i in range(half)]
        return [x / s * (1 - k) + x * k for x, k in zip(f, stays)], 0.1 * math.log(s) + 1
    return f, 1.0


def _slopes(heads):
    return [2 ** (-8 * (h + 1) / heads) for h in range(heads)]


def _positions(c):
    """Place in the sequence of every row of a ring's tensors."""
    n, ranks = c["tokens"], c["ranks"]
    if not ranks:
        return list(range(n))
    half = n // (2 * ranks)
    return [x for r in range(ranks) for at in (r, 2 * ranks - 1 - r) for x in range(at * half, (at + 1) * half)]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, hkv, d = TORCH[c["dtype"]], c["page"], c["kv_heads"], c["dim"]
    s = {"case": c}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    if "turned" in c:
        f, s["factor"] = _frequencies(c)
        s["frequencies"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        if own:
            from ringattention_amd.rotary import Rotary
            s["rotary"] = Rotary(d, c["turned"], base=BASE, interleaved=c["interleaved"], scaling=c["scaling"] or None, factor=c["spread"], trained=TRAINED, dtype=c["dtype"])
    if c["op"] == "rotate":
        s["positions"] = ints(_positions(c))
        s["q"], s["k"] = normal(1, c["heads"], c["tokens"], d), normal(1, hkv, c["tokens"], d)
        if own:
            s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s
    lens, news = _ints(c["lens"]), _ints(c["news"])
    if c["op"] in ("fork", "compact"):
        return _prepare_pages(c, s, gen, normal, ints, lens)
    pages = [-(-n // page) for n in lens]
    order = torch.randperm(sum(pages), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    s["table"] = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        s["table"][b, :n] = order[at:at + n]
        at += n
    s["lens"], T = ints(lens), sum(news)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s["starts"] = ints(starts)
    s["q"] = normal(T, c["heads"], d)
    s["k_cache"], s["v_cache"] = normal(at, hkv, page, d), normal(at, hkv, page, d)
    if own:
        from ringattention_amd import paged
    if c["op"] == "append":
        s["k"], s["v"] = normal(T, hkv, d), normal(T, hkv, d)
        if own:
            s["plan"] = paged.PagedAttention(c["heads"], d, kv_heads=hkv, dtype=c["dtype"], page_size=page, max_batch=len(lens), max_tokens=max(1, T))
            s["q_out"] = torch.empty_like(s["q"])
        return s
    # queries somewhat aligned with keys, so that scores reach the cap
    s["q"] *= 2
    s["slopes"] = torch.tensor(_slopes(c["heads"]), dtype=torch.float32, device="cuda") if c["slopes"] else None
    s["prefix"] = ints([min(n, c["prefix"] + b % 3) for b, n in enumerate(lens)]) if c["prefix"] else None
    s["first"] = None
    if c["docs"]:
        places = torch.cat([torch.arange(n - m, n, dtype=torch.int32) for n, m in zip(lens, news)]).to("cuda")
        s["first"] = places // c["docs"] * c["docs"]
    if c["op"] == "weights":
        s["scores"] = torch.relu(torch.randn((at, hkv, page), generator=gen, device="cuda"))
        s["lse"] = _plain_attend(s)[1]
    if own:
        s["plan"] = paged.PagedAttention(c["heads"], d, kv_heads=hkv, dtype=c["dtype"], page_size=page, max_batch=len(lens), max_tokens=max(1, T),
                                         window=c["window"], sinks=c["sinks"], softcap=c["cap"], slopes=s["slopes"])
        if c["op"] == "attend":
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(c["heads"], T, dtype=torch.float32, device="cuda")
    return s


def _page_plan(c):
    """Of a fork or compact case, the rows' page counts, entries of a row of the table, pages of the pool."""
    lens = _ints(c["lens"])
    counts = [-(-n // c["page"]) for n in lens]
    if c["op"] == "fork":   # what the first rows of the groups have, and as much for rows that begin anew
        used = sum(counts)
        return counts, max(counts) + 1, used + len(lens) + 1
    return counts, max(counts) + 1, sum(counts) * c["spare"] // 2 + 1


def _prepare_pages(c, s, gen, normal, ints, lens):
    counts, entries, pages = _page_plan(c)
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    s["table"] = torch.full((len(lens), entries), -1, dtype=torch.int32, device="cuda")
    s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
    s["lens"] = ints(lens)
    at = 0
    for b, n in enumerate(counts):
        s["table"][b, :n] = order[at:at + n]
        at += n
    s["refs"][order[:at].long()] = 1
    s["k_cache"], s["v_cache"] = normal(pages, c["kv_heads"], c["page"], c["dim"]), normal(pages, c["kv_heads"], c["page"], c["dim"])
    if c["op"] == "fork":   # the rows of a group become forks of its first, but for its last, which begins anew
        g = c["groups"]
        parents = [b - b % g for b in range(len(lens))]
        add = [0 if b % g == 0 else 1 for b in range(len(lens))]
        for b in range(g - 1, len(lens), g):
            if g > 2:
                parents[b], add[b] = -1, max(1, lens[b] // 2)
        s["parents"], s["add"] = ints(parents), ints(add)
    s["before"] = [s[x].clone() for x in ("table", "refs", "lens")]
    if own:
        from ringattention_amd import paged
        s["pool"] = paged.PagePool(pages, len(lens), entries, page_size=c["page"])
        for mine, given in zip((s["pool"].page_table, s["pool"].refs, s["pool"].lens), s["before"]):
            mine.copy_(given)
        s["short"] = torch.empty(len(lens), dtype=torch.int32, device="cuda")
        s["used"] = torch.empty(1, dtype=torch.int32, device="cuda")
    return s


# ---- plain forms: rotary positions

def _turn(x, angles, c, factor):
    """x [..., dim] in 32 bits, angles [..., pairs] in 64 bits that go with it."""
    cos, sin = (torch.cos(angles) * factor).float(), (torch.sin(angles) * factor).float()
    if c.get("inverse"):
        sin = -sin
    r = c["turned"]
    t = x[..., :r]
    a, b = (t[..., 0::2], t[..., 1::2]) if c["interleaved"] else (t[..., :r // 2], t[..., r // 2:])
    p, q = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((p, q), dim=-1).flatten(-2) if c["interleaved"] else torch.cat((p, q), dim=-1)
    return torch.cat((y, x[..., r:]), dim=-1)


def _plain_rotate(s):
    angles = s["positions"].double()[:, None] * s["frequencies"]
    return tuple(_turn(s[x].float(), angles, s["case"], s["factor"]).to(s[x].dtype) for x in ("q", "k"))


def _token_places(s, T):
    """Of every new token: its sequence, its number among that one's new tokens, its position in the sequence."""
    starts = s["starts"].long()
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(starts, t, right=True) - 1
    i = t - starts[b]
    return b, i, s["lens"].long()[b] - (starts[b + 1] - starts[b]) + i


def _plain_append(s):
    c = s["case"]
    b, _, place = _token_places(s, s["q"].shape[0])
    angles = (place.double()[:, None] * s["frequencies"])[:, None]
    pages = s["table"].long()[b, place // c["page"]]
    s["k_cache"][pages, :, place % c["page"]] = _turn(s["k"].float(), angles, c, s["factor"]).to(s["k"].dtype)
    s["v_cache"][pages, :, place % c["page"]] = s["v"]
    return _turn(s["q"].float(), angles, c, s["factor"]).to(s["q"].dtype), s["k_cache"], s["v_cache"]


# ---- plain forms: attention

def _gathered(cache, table):
    """The sequences' rows of a cache in 32 bits, [batch, kv_heads, keys, dim]."""
    x = cache[table.long().clamp(min=0)].float()
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _seen(c, place, key, prefix, first):
    """Which keys a token at `place` sees."""
    seen = key <= place
    near = torch.ones_like(seen)
    if c["window"]:
        near = key > place - c["window"]
    if first is not None:
        near = near & (key >= first)
    if c["window"] and c["sinks"]:
        near = near | (key < c["sinks"])
    seen = seen & near
    return seen | (key < prefix) if prefix is not None else seen


def _padded_scores(s):
    """(scores [batch, kv_heads, new tokens x heads of a group, keys] in 32 bits with -inf where a key is hidden, sequence and number of every token)"""
    c = s["case"]
    hkv, group, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    T = s["q"].shape[0]
    b, i, _ = _token_places(s, T)
    most = max(_ints(c["news"]))
    starts, lens = s["starts"].long(), s["lens"].long()
    n = starts[1:] - starts[:-1]
    at = torch.arange(most, device="cuda")
    tokens = (starts[:-1, None] + torch.minimum(at[None, :], (n - 1).clamp(min=0)[:, None])).clamp(max=T - 1)
    q = s["q"][tokens].float().reshape(len(lens), most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(len(lens), hkv, most * group, d)
    x = torch.matmul(q, _gathered(s["k_cache"], s["table"]).transpose(2, 3)).mul_(1 / math.sqrt(d))
    del q
    if c["cap"]:
        x.div_(c["cap"]).tanh_().mul_(c["cap"])
    key = torch.arange(x.shape[3], device="cuda")
    place = ((lens - n)[:, None] + at[None, :])[:, :, None]   # [batch, new tokens, 1]
    seen = _seen(c, place, key, None if s["prefix"] is None else s["prefix"].long()[:, None, None], None if s["first"] is None else s["first"].long()[tokens][:, :, None])
    seen &= (key < lens[:, None, None]) & (at[None, :] < n[:, None])[:, :, None]
    by_head = x.view(len(lens), hkv, most, group, x.shape[3])
    if c["slopes"]:
        far = (place - key).abs().float()   # [batch, new tokens, keys]
        for h in range(c["heads"]):
            by_head[:, h // group, :, h % group].addcmul_(far, -s["slopes"][h])
    by_head.masked_fill_(~seen[:, None, :, None], -math.inf)
    return x, b, i


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


# ---- plain forms: pages

def _count(refs, pages, by):
    """refs with `by` added for every page of a list (-1: none)."""
    refs.index_add_(0, pages.reshape(-1).long().clamp(min=0), torch.where(pages.reshape(-1) >= 0, by, 0).to(refs.dtype))


def _plain_fork(s):
    """New rows share what they keep of their parents' pages.  Rows that grow take pages of the pool, lowest first, in the order of the rows
    while there are enough; a shared page that is going to be written is copied."""
    page, (R, E) = s["case"]["page"], s["table"].shape
    table, refs, parents = s["table"].long(), s["refs"], s["parents"].long()
    had = torch.where(parents >= 0, s["lens"].long()[parents.clamp(min=0)], 0)
    want = (had + s["add"].long()).clamp(min=0)
    entry = torch.arange(E, device="cuda")
    kept = (torch.minimum(had, want) + page - 1) // page
    made = torch.where((entry < kept[:, None]) & (parents >= 0)[:, None], table[parents.clamp(min=0)], -1)
    _count(refs, table, -1)
    _count(refs, made, 1)
    part = (had // page).clamp(max=E - 1)   # the entry that is written on, where it is not full
    torn = made.gather(1, part[:, None])[:, 0]
    copies = (want > had) & (had % page != 0) & (torn >= 0) & (refs[torn.clamp(min=0)] > 1)
    need = (want + page - 1) // page - kept + copies.long()
    fits = want <= E * page
    need = torch.where(fits, need, 0)
    free = refs == 0
    upto = need.cumsum(0)
    grows = fits & (upto <= free.sum())
    short = (want > had) & ~grows
    copies &= grows
    now = torch.where(short, had, want)
    pool = torch.nonzero(free)[:, 0]
    first = kept - copies.long()   # the first entry that a row takes from the pool
    takes = grows[:, None] & (entry >= first[:, None]) & (entry < ((want + page - 1) // page)[:, None])
    at = (upto - need)[:, None] + entry - first[:, None]
    taken = pool[torch.where(takes, at, 0)] if pool.numel() else at   # (nothing is taken of an empty pool)
    source, target = torn[copies], taken.gather(1, part[:, None])[:, 0][copies]
    s["k_cache"][target] = s["k_cache"][source]
    s["v_cache"][target] = s["v_cache"][source]
    _count(refs, torch.where(copies, torn, -1), -1)
    made = torch.where(takes, taken, made)
    _count(refs, torch.where(takes, taken, -1), 1)
    s["table"].copy_(made)
    s["lens"].copy_(now)
    return s["table"], s["lens"], refs, short.to(torch.int32), s["k_cache"], s["v_cache"]


def _plain_compact(s):
    refs, pages = s["refs"], s["refs"].shape[0]
    used = refs > 0
    n = used.sum()
    place = torch.arange(pages, device="cuda")
    source, target = torch.nonzero(used & (place >= n))[:, 0], torch.nonzero(~used & (place < n))[:, 0]
    s["k_cache"][target] = s["k_cache"][source]
    s["v_cache"][target] = s["v_cache"][source]
    moved = place.clone()
    moved[source] = target
    refs[target] = refs[source]
    refs[source] = 0
    table = s["table"].long()
    s["table"].copy_(torch.where(table >= 0, moved[table.clamp(min=0)], table))
    return s["table"], refs, n.to(torch.int32).reshape(1), s["k_cache"], s["v_cache"]


def run(s):
    c = s["case"]
    op = c["op"]
    if op in ("fork", "compact"):   # the rows as they were before: a step of a loop whose other steps had them become so
        state = (s["pool"].page_table, s["pool"].refs, s["pool"].lens) if own else (s["table"], s["refs"], s["lens"])
        for now, before in zip(state, s["before"]):
            now.copy_(before)
        if not own:
            return _plain_fork(s) if op == "fork" else _plain_compact(s)
        pool, cache = s["pool"], (s["k_cache"], s["v_cache"])
        if op == "fork":
            pool.update(*cache, parents=s["parents"], add=s["add"], short=s["short"])
            return (pool.page_table, pool.lens, pool.refs, s["short"]) + cache
        pool.compact(*cache, used=s["used"])
        return (pool.page_table, pool.refs, s["used"]) + cache
    if not own:
        return {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend, "weights": _plain_weights}[op](s)
    if op == "rotate":
        return s["rotary"].apply(s["q"], s["k"], s["positions"], s["q_out"], s["k_out"], inverse=c["inverse"])
    plan, seqs = s["plan"], (s["table"], s["lens"], s["starts"])
    if op == "append":
        plan.append_rotary(s["rotary"], s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], *seqs, q_out=s["q_out"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    if op == "attend":
        return plan.forward(s["q"], s["k_cache"], s["v_cache"], *seqs, s["out"], s["lse"], prefix_lens=s["prefix"], first_keys=s["first"])
    return plan.weights(s["q"], s["lse"], s["k_cache"], *seqs, s["scores"], prefix_lens=s["prefix"], first_keys=s["first"])


# ---- what a pass cannot do without

def _visible(c, length, new, b):
    """Visible (query, key) pairs of a head of a sequence, and its keys that some query sees."""
    prefix = min(length, c["prefix"] + b % 3) if c["prefix"] else 0
    pairs, low_all = 0, length
    window, sinks = c["window"] or length, c["sinks"] if c["window"] else 0
    for p in range(length - new, length):
        low = max(p + 1 - window, p // c["docs"] * c["docs"] if c["docs"] else 0, 0)
        front = max(prefix, min(sinks, p + 1))   # [0, front) and [low, p] are seen
        pairs += front + max(0, p + 1 - max(low, front))
        low_all = min(low_all, low)
    front = max(prefix, min(sinks, length))
    return pairs, min(length, front + max(0, length - max(low_all, front))) if new else 0


def work(case):
    c = case
    hkv, H, d = c["kv_heads"], c["heads"], c["dim"]
    if c["op"] == "rotate":   # Q and K read and written; two products and a sum for a turned column
        return {"bytes": c["tokens"] * (H + hkv) * d * 4 + c["tokens"] * 4, "flops": 3 * c["tokens"] * (H + hkv) * c["turned"]}
    lens, news = _ints(c["lens"]), _ints(c["news"])
    if c["op"] == "append":   # Q, K and V read and written
        return {"bytes": sum(news) * (H + 2 * hkv) * d * 4, "flops": 3 * sum(news) * (H + hkv) * c["turned"]}
    if c["op"] == "fork":   # old and new entries, counts of the pages they name; a page of K and V read and written for a row that leaves one unfull
        counts, entries, _ = _page_plan(c)
        g, page = c["groups"], hkv * c["page"] * d * 4
        anew = [g > 2 and b % g == g - 1 for b in range(len(lens))]
        copied = sum(1 for b, n in enumerate(lens) if b % g and not anew[b] and n % c["page"])
        return {"bytes": sum(counts) * 2 * 12 + copied * 2 * page, "flops": 0}
    if c["op"] == "compact":   # counts, entries read and written; pages of K and V that lie behind the ones that stay, about that share of them
        counts, _, pages = _page_plan(c)
        moved = sum(counts) * (1 - sum(counts) / pages)
        return {"bytes": int(pages * 8 + sum(counts) * 8 + moved * 2 * hkv * c["page"] * d * 4), "flops": 0}
    both = [_visible(c, n, m, b) for b, (n, m) in enumerate(zip(lens, news))]
    pairs, keys = sum(x[0] for x in both), sum(x[1] for x in both)
    if c["op"] == "attend":   # K and V that are seen, Q and O, LSE
        return {"bytes": keys * hkv * d * 4 + sum(news) * H * (4 * d + 4), "flops": 4 * d * H * pairs}
    # weights: K, Q and LSE; a score of every key read and written
    return {"bytes": keys * hkv * (2 * d + 8) + sum(news) * H * (2 * d + 4), "flops": 2 * d * H * pairs}


# ---- the definitions in 64 bits, row by row

def exact(case, seed):
    """Rotary positions as products of complex numbers; attention sequence by sequence and head by head, over rows of a cache by (page, slot)."""
    c = case
    if c["op"] in ("fork", "compact"):
        return None   # pages are counted and copied, nothing is computed
    s = prepare(case, seed)
    lens, news, page = _ints(c["lens"]), _ints(c["news"]), c["page"]
    hkv, group, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]

    def turned(x, places):   # x [tokens, heads, dim]
        x = x.double()
        for i in range(c["turned"] // 2):
            a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + c["turned"] // 2)
            z = torch.complex(x[..., a], x[..., b])
            angle = places.double() * float(s["frequencies"][i]) * (-1 if c.get("inverse") else 1)
            z = z * torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None]
            x[..., a], x[..., b] = z.real, z.imag
        return x

    if c["op"] == "rotate":
        return tuple(turned(s[x][0].transpose(0, 1), s["positions"]).transpose(0, 1)[None] for x in ("q", "k"))
    place = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, news)])
    of = torch.cat([torch.full((m,), b, device="cuda") for b, m in enumerate(news)])
    if c["op"] == "append":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        pages = s["table"][of, place // page].long()
        k[pages, :, place % page] = turned(s["k"], place)
        v[pages, :, place % page] = s["v"].double()
        return turned(s["q"], place), k, v
    if sum(n * m for n, m in zip(lens, news)) * c["heads"] * d > 1.5e12:
        return None   # (64-bit products of some minute)

    def rows(cache, b, h, n):
        pages = s["table"][b, :-(-n // page)].long()
        return cache[pages, h].reshape(-1, *cache.shape[3:])[:n]

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(c["heads"], s["q"].shape[0], dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if c["op"] == "weights" else None
    for b, (n, m) in enumerate(zip(lens, news)):
        at = int(s["starts"][b])
        key = torch.arange(n, device="cuda")[None, :]
        prefix = min(n, c["prefix"] + b % 3) if c["prefix"] else 0
        for h in range(hkv if m else 0):
            k = rows(s["k_cache"], b, h, n).double()
            v = rows(s["v_cache"], b, h, n).double() if c["op"] == "attend" else None
            drawn = torch.zeros(n, dtype=torch.float64, device="cuda")
            for i in range(0, m, 512):
                t = slice(at + i, at + min(m, i + 512))
                p = place[t][:, None]
                hidden = key > p
                if c["docs"]:
                    other = key < torch.div(p, c["docs"], rounding_mode="floor") * c["docs"]
                    hidden = hidden | (other & (key >= (c["sinks"] if c["window"] else 0)))
                if c["window"]:
                    hidden = hidden | ((p - key >= c["window"]) & (key >= c["sinks"]))
                hidden = hidden & (key >= prefix)
                for g in range(h * group, (h + 1) * group):
                    x = s["q"][t, g].double() @ k.t() / d ** 0.5
                    if c["cap"]:
                        x = c["cap"] * torch.tanh(x / c["cap"])
                    if c["slopes"]:
                        x = x - float(s["slopes"][g]) * (p - key).abs()
                    x = x.masked_fill(hidden, -math.inf)
                    if c["op"] == "attend":
                        z = torch.logsumexp(x, dim=1)
                        lse[g, t] = z
                        out[t, g] = torch.exp(x - z[:, None]) @ v
                    else:
                        drawn += torch.exp(x - s["lse"][g, t].double()[:, None]).sum(dim=0)
            if scores is not None:
                j = torch.arange(n, device="cuda")
                scores[s["table"][b].long()[j // page], h, j % page] += drawn
    return (out, lse) if c["op"] == "attend" else scores
