"""Q, K and V of one fused product on their way into the cache, Q turned in place or elsewhere: the layouts whose rows lie between each other."""
import pytest
import torch

import paged_reference as ref
from ringattention_amd import paged
from ringattention_amd.rotary import Rotary

pytestmark = pytest.mark.gpu


def fused(layout, T, heads, kv, d, dtype):
    """(q, k, v), views of one tensor, [tokens, heads, d]."""
    g = torch.Generator(device="cuda").manual_seed(heads + kv)
    make = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)   # noqa: E731
    if layout == "a token's heads one behind the other":
        x = make(T, heads + 2 * kv, d)
        return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if layout == "with room between":
        x = make(T, heads + 2 * kv + 3, d)
        return x[:, 1:1 + heads], x[:, heads + 1:heads + 1 + kv], x[:, heads + 3 + kv:]
    if layout == "head by head":
        x = make(heads + 2 * kv, T, d).transpose(0, 1)
        return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    x = make(T, heads, 3, d) if layout == "a head's three rows" else make(heads, T, 3, d).transpose(0, 1)
    return x[:, :, 0], x[:, :, 1], x[:, :, 2]


@pytest.mark.parametrize("layout,heads,kv", [("a token's heads one behind the other", 8, 2), ("a token's heads one behind the other", 3, 3), ("with room between", 8, 4),
                                             ("head by head", 4, 2), ("a head's three rows", 4, 4), ("a head's three rows, head by head", 2, 2), ("a head's three rows", 1, 1)])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("news", [[1], [9, 1, 30]])
def test_rows_between_each_other(layout, heads, kv, in_place, news):
    d, dtype = 64, torch.bfloat16
    c = ref.Case(dtype="bf16", dim=d, heads=heads, kv_heads=kv, lens=[40 + n for n in news], news=news, spare=0.0)
    r = Rotary(d, dtype="bf16")
    plan = paged.PagedAttention(heads, d, kv_heads=kv, dtype="bf16", page_size=16, max_batch=len(news), max_tokens=c.tokens)
    q, k, v = fused(layout, c.tokens, heads, kv, d, dtype)
    seqs = (c.table.cuda(), c.kv_lens().cuda(), c.starts.cuda())
    apart = [x.contiguous().clone() for x in (q, k, v)]
    want = [c.k.cuda(), c.v.cuda()]
    want_q = plan.append_rotary(r, *apart, *want, *seqs)
    got = [c.k.cuda(), c.v.cuda()]
    out = q if in_place else torch.empty_like(q)
    assert plan.append_rotary(r, q, k, v, *got, *seqs, q_out=out) is out
    assert torch.equal(out, want_q) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(k, apart[1]) and torch.equal(v, apart[2])


def test_on_each_other_is_refused():
    c = ref.Case(dtype="bf16", dim=64, heads=4, kv_heads=4, lens=[9], news=[9], spare=0.0)
    r = Rotary(64, dtype="bf16")
    plan = paged.PagedAttention(4, 64, dtype="bf16", page_size=16, max_batch=1, max_tokens=9)
    k, v = (torch.zeros(9, 4, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for out in (k, v):
        with pytest.raises(RuntimeError):
            plan.append_rotary(r, c.q.cuda(), k, v, c.k.cuda(), c.v.cuda(), c.table.cuda(), c.kv_lens().cuda(), c.starts.cuda(), q_out=out)


@pytest.mark.parametrize("batch", [65, 1000, 4096])
def test_as_many_sequences_as_a_plan_takes(batch):
    """Single tokens, sequences without any and some with several, on a stream: the same bits as turning first and appending then."""
    news = [(0, 1, 1, 1, 3, 1, 0)[i % 7] for i in range(batch)]
    lens = [max(1, n) + (i * 29) % 40 for i, n in enumerate(news)]
    c = ref.Case(dtype="fp16", dim=64, heads=2, kv_heads=1, lens=lens, news=news, spare=0.0, extra_rows=2)
    r = Rotary(64, dtype="fp16", interleaved=True)
    plan = paged.PagedAttention(2, 64, kv_heads=1, dtype="fp16", page_size=16, max_batch=batch, max_tokens=c.tokens)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((c.tokens, 1, 64), generator=g, device="cuda").half() for _ in range(2))
    q, seqs = c.q.cuda(), (c.table.cuda(), c.kv_lens().cuda(), c.starts.cuda())
    pos = torch.tensor([n - m + i for n, m in zip(lens, news) for i in range(m)] + [0, 0], dtype=torch.int32).cuda()
    want = [c.k.cuda(), c.v.cuda()]
    want_q, turned = r.apply(q, k, pos)
    plan.append(turned, v, *want, *seqs)
    got, out = [c.k.cuda(), c.v.cuda()], torch.full_like(q, 3.0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    plan.append_rotary(r, q, k, v, *got, *seqs, q_out=out, stream=stream)
    stream.synchronize()
    assert torch.equal(out[:-2], want_q[:-2]) and (out[-2:] == 3).all() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
