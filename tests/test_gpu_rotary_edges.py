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
