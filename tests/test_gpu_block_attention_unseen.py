"""ress_amd.block_attention: keys that a row does not see, and such as weigh nothing for it, leave its gradient alone, however
large they are."""

import pytest
import torch

import ress_amd as ress
from attention_reference import visible
from attention_rounded import attention, off

pytestmark = pytest.mark.gpu


def make(H, Tq, Tk, D, dt, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(1, H, T, D, generator=g) for T in (Tq, Tk, Tk, Tq))
    return [t.to(dev, dt) for t in (q, k + 0.3, v + 0.5, 0.1 * do)]


def run(q, k, v, do, **kw):
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = ress.block_attention(*leaves, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, do)]


# calls of few probabilities, whole ones, and such as are cut into parts
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Tq,Tk", [(2, 300, 300), (2, 511, 511), (2, 100, 1400), (1, 1400, 1400), (40, 1340, 1340)])
def test_long_keys_above_the_diagonal(dev, dt, D, H, Tq, Tk):
    """Rows before the last 20 give the same bits whatever finite keys stand in the last 20 places."""
    q, k, v, do = make(H, Tq, Tk, D, dt, dev)
    want = run(q, k, v, do, causal=True)
    k[:, :, Tk - 20:] *= 1000.0
    got = run(q, k, v, do, causal=True)
    for i in (0, 1):
        assert torch.equal(got[i][:, :, :Tq - 20], want[i][:, :, :Tq - 20])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Tq,Tk", [(2, 200, 1025), (2, 200, 2049), (48, 1300, 705), (1, 130, 20000)])
def test_long_keys_that_weigh_nothing(dev, dt, D, H, Tq, Tk):
    """The first and the last key are 200 long and have probabilities below 2^-20 of the others' (-200 q0 / sqrt(D), q0 = 1.5): dQ's error is that of the
    same roundings in 64 bits. Errors of the same kind over 130 rows or more of 64 values: their norms differ by less than half."""
    q, k, v, do = make(H, Tq, Tk, D, dt, dev)
    q[..., 0] = 1.5
    for j in (0, -1):
        k[:, :, j] = 0.0
        k[:, :, j, 0] = -200.0
    got = run(q, k, v, do)
    see = visible(1, 1, Tq, Tk)
    worst, like = [], []
    for h in range(0, H, 4):  # four heads at a time, for the memory
        part = [t[:, h:h + 4] for t in (q, k, v)]
        exact = attention(*part, see, do[:, h:h + 4])[1]
        worst.append(off(got[1][:, h:h + 4], exact))
        like.append(off(attention(*part, see, do[:, h:h + 4], dt)[1], exact))
    assert max(worst) <= 1.5 * max(like), (worst, like)
