"""Arguments that get no gradient are refused where one is asked of them."""

import pytest
import torch

import ress_amd as ress

pytestmark = pytest.mark.gpu


def test_a_scale_with_a_gradient(dev):
    q = torch.randn(1, 2, 8, 64, device=dev).bfloat16()
    scale = torch.tensor(0.1, requires_grad=True)
    want = ress.block_attention(q, q, q, scale=0.1)
    with pytest.raises(ValueError, match="scale gets no gradient"):
        ress.block_attention(q, q, q, scale=scale)
    assert torch.equal(ress.block_attention(q, q, q, scale=scale.detach()), want)
    with torch.no_grad():
        assert torch.equal(ress.block_attention(q, q, q, scale=scale), want)


def test_a_table_with_a_gradient(dev):
    x, pos = torch.randn(1, 2, 8, 64, device=dev).bfloat16(), torch.arange(8, device=dev)
    values = ress.RotaryTable(64, 8, axes=1, device=dev).table
    want = ress.rotate(x, pos, ress.RotaryTable.from_table(values, 64, 1))
    rope = ress.RotaryTable.from_table(values.clone().requires_grad_(), 64, 1)
    with pytest.raises(ValueError, match="table gets no gradient"):
        ress.rotate(x, pos, rope)
    with torch.no_grad():
        assert torch.equal(ress.rotate(x, pos, rope), want)
