"""ress_amd.block_attention at its ends: no query heads, more rows than one join could take."""

import pytest
import torch

import ress_amd as ress
from attention_reference import visible
from attention_rounded import attention, off

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mapped", [False, True])
@pytest.mark.parametrize("Tq,Tk", [(5, 70), (0, 70), (5, 0), (300, 2000)])
def test_no_query_heads(dev, dt, mapped, Tq, Tk):
    """An empty output, and zero gradients of the keys and values that nothing has seen."""
    q = torch.empty(2, 0, Tq, 64, dtype=dt, device=dev, requires_grad=True)
    junk = torch.full((2, 2, Tk, 64), 3.0, dtype=dt, device=dev)  # memory that the gradients may get
    k, v = (torch.ones(2, 2, Tk, 64, dtype=dt, device=dev, requires_grad=True) for _ in range(2))
    m = torch.ones(2, 1, -(-Tq // 128), -(-Tk // 64), dtype=torch.bool, device=dev).expand(2, 1, -1, -1)[:, :0] if mapped else None
    out = ress.block_attention(q, k, v, block_map=m)
    assert out.shape == q.shape
    del junk
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.empty_like(out))
    assert dq.shape == q.shape and dk.shape == k.shape and (dk == 0).all() and (dv == 0).all()
