"""Forward-mode derivatives, which the operators with a backward pass do not have, are refused and not dropped."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import ress_amd as ress
from ress_amd import differentiable as df
from ress_amd.aggregator import Block, RoPE2D


@pytest.mark.parametrize("enabled", [True, False])
def test_a_tangent_is_seen(enabled):
    x, y = torch.randn(2, 8), torch.randn(2, 8)
    with torch.set_grad_enabled(enabled), fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for given in ((dual,), (y, dual), (None, y, dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                df._differentiates(*given)
        assert not df._differentiates(x, None, y)
    assert not df._differentiates(x)


@pytest.mark.gpu
def test_the_operators(dev):
    def t(*shape):
        return torch.randn(*shape, device=dev).bfloat16()

    rope = ress.RotaryTable(64, 8, axes=1, device=dev)
    q, pos, w = t(1, 2, 8, 64), torch.arange(8, device=dev), t(64)
    calls = [lambda x: ress.block_attention(x, q, q), lambda x: ress.block_attention(q, q, x), lambda x: ress.layer_norm(x),
             lambda x: ress.add_layer_norm(q, x), lambda x: ress.rotate(x, pos, rope), lambda x: ress.rotate((q, x), pos, rope)]
    for call in calls:
        want = call(q)
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(fw.make_dual(q.clone(), torch.ones_like(q)))
            again = call(q)
        for a, b in zip((want,) if torch.is_tensor(want) else want, (again,) if torch.is_tensor(again) else again):
            assert torch.equal(a, b)
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ress.layer_norm(q, fw.make_dual(w, torch.ones_like(w)))


@pytest.mark.gpu
def test_a_frozen_block(dev):
    """A block without trainable parameters under enable_gradients: a tangent that torch's modules would hand on is refused."""
    block = Block(128, 2, 2.0, RoPE2D()).to(dev, torch.bfloat16).requires_grad_(False)
    ress.enable_gradients(block)
    x = torch.randn(1, 6, 128, device=dev).bfloat16()
    pos = torch.zeros(1, 6, 2, dtype=torch.int64, device=dev)
    block(x, pos)
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        block(fw.make_dual(x, torch.ones_like(x)), pos)
