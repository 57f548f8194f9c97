"""ress_amd.block_attention over few terms a result in many heads: more than 2^18 probabilities, so rounded ones."""

import pytest
import torch

import ress_amd as ress
from attention_reference import visible
from attention_rounded import attention, off

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,u", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hq,Hk,Tq,Tk", [(32, 32, 32, 1, 300), (32, 32, 4, 1, 300), (400, 128, 128, 1, 6), (400, 64, 64, 12, 1), (8, 64, 64, 5, 129)])
def test_few_terms_a_result(dev, dt, u, D, B, Hq, Hk, Tq, Tk):
    """Each output at the error of the same roundings, and below u: three roundings (P's, dS's or delta's, the result's) of at most u, u / sqrt(3)
    rms each, independent of one another and however many terms a result has."""
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(B, H, T, D, generator=g).to(dev, dt) for H, T in ((Hq, Tq), (Hk, Tk), (Hk, Tk), (Hq, Tq)))
    assert B * Hq * Tq * Tk > 1 << 18
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ress.block_attention(*leaves)
    got = (out, *torch.autograd.grad(out, leaves, do))
    see = visible(1, 1, Tq, Tk)
    exact, like = attention(q, k, v, see, do), attention(q, k, v, see, do, dt)
    for name, x, y, z in zip(("out", "dq", "dk", "dv"), got, exact, like):
        if Tk == 1 and name in ("dq", "dk"):
            # one key: P is 1 and dS 0 but for what 32 bits leave of dP - delta, 2^-20 of its terms' size
            size = 0.125 * (do.float().norm(dim=-1).max() * v.float().norm(dim=-1).max() * max(q.abs().max(), k.abs().max())).item()
            assert x.abs().max().item() <= 2.0 ** -20 * size * Tq * (Hq // Hk)
        else:
            assert off(x, y) <= min(u, 1.25 * off(z, y)), name
