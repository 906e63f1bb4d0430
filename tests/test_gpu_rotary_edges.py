"""Rotary positions of tensors that have nothing in one dimension."""
import pytest
import torch

from ringattention_amd.rotary import Rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,none", [((1, 3, 7, 64), (1, 0, 7, 64)), ((2, 1, 5, 64), (2, 0, 5, 64)), ((7, 3, 64), (7, 0, 64))])
def test_a_tensor_of_no_heads_leaves_the_other_its_turn(shape, none):
    r = Rotary(64, dtype="bf16")
    x = torch.randn(shape, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    empty = torch.empty(none, dtype=torch.bfloat16, device="cuda")
    want = r.apply(x)[0]
    for q, k, of in ((x, empty, 0), (empty, x, 1)):
        out = [torch.full_like(q, 5.0), torch.full_like(k, 5.0)]
        r.apply(q, k, q_out=out[0], k_out=out[1])
        assert torch.equal(out[of], want) and torch.equal(r.apply(q, k)[of], want)
    assert r.apply(empty)[0].shape == empty.shape and r.apply(empty, empty)[1].shape == empty.shape


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("heads,kv,batch,tokens", [(8, 2, 1, 9), (3, 3, 2, 7), (4, 1, 3, 1), (1, 1, 2, 5), (1, 4, 2, 6)])
@pytest.mark.parametrize("layout", ["a token's heads", "head by head", "batches within tokens", "a head's three rows"])
def test_q_and_k_between_each_other(layout, heads, kv, batch, tokens, in_place):
    """Views of one fused product."""
    r = Rotary(64, dtype="fp16")
    g = torch.Generator().manual_seed(heads + kv)
    make = lambda *shape: torch.randn(shape, generator=g).half().cuda()   # noqa: E731
    if layout == "a token's heads":
        x = make(batch, tokens, heads + 2 * kv, 64).transpose(1, 2)
    elif layout == "head by head":
        x = make(batch, heads + 2 * kv, tokens, 64)
    elif layout == "batches within tokens":
        x = make(tokens, batch, heads + 2 * kv, 64).permute(1, 2, 0, 3)
    else:
        kv = heads
        x = make(batch, tokens, heads, 3, 64).permute(3, 0, 2, 1, 4)
        q, k = x[0], x[1]
    if layout != "a head's three rows":
        q, k = x[:, :heads], x[:, heads:heads + kv]
    want = [r.apply(t.contiguous())[0] for t in (q, k)]
    rest = (x[2] if layout == "a head's three rows" else x[:, heads + kv:]).clone()
    got = r.apply(q, k, q_out=q, k_out=k) if in_place else r.apply(q, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(rest, x[2] if layout == "a head's three rows" else x[:, heads + kv:])


def test_q_and_k_on_each_other_are_refused():
    r = Rotary(64, dtype="fp16")
    x = torch.zeros(2, 5, 12, 64, dtype=torch.float16, device="cuda").transpose(1, 2)
    for q, k in ((x[:, :8], x[:, 7:9]), (x[:, 1:9], x[:, :2]), (x[:, :8, :4], x[:, :2, 1:])):
        with pytest.raises(RuntimeError):
            r.apply(q, k, q_out=q, k_out=k)
