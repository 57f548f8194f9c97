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


def test_very_many_rows(dev):
    """64 heads of 2^20 rows over 64 keys, and all of their gradients: the same bits as a head by itself, dK and dV at the roundings' error."""
    g = torch.Generator().manual_seed(0)
    q, do = (torch.randn(1, 1, 1 << 20, 64, generator=g).to(dev, torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(1, 64, 64, 64, generator=g).to(dev, torch.bfloat16).requires_grad_() for _ in range(2))
    every = q.expand(-1, 64, -1, -1).requires_grad_()
    out = ress.block_attention(every, k, v)
    dq, dk, dv = torch.autograd.grad(out, (every, k, v), do.expand(-1, 64, -1, -1))
    for h in (0, 37, 63):
        alone = [t.detach().clone().requires_grad_() for t in (q, k[:, h:h + 1], v[:, h:h + 1])]
        one = ress.block_attention(*alone)
        assert torch.equal(one[0, 0], out[0, h]) and torch.equal(torch.autograd.grad(one, alone[0], do)[0][0, 0], dq[0, h])
    del out, dq
    q, k, v = q.detach(), k.detach()[:, 37:38], v.detach()[:, 37:38]
    see = visible(1, 1, 1, 64).expand(1, 1, 1 << 20, 64)
    exact = attention(q, k, v, see, do)
    for n, x in ((2, dk), (3, dv)):
        # three roundings of 2^-8 / sqrt(3) rms, and sums of 2^20 terms in 32 bits, 2^-24 of a sum that is 2^10 terms' size at most: 2^-14 of a term's
        assert off(x[:, 37:38], exact[n]) <= 2.0 ** -8 + 2.0 ** -10
