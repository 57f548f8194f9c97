"""ress_amd.block_attention in fp16: what a row or a key does not see, and what other rows and keys see, takes no precision from its
gradients, however large it is."""

import pytest
import torch

import ress_amd as ress
from attention_reference import visible
from attention_rounded import attention, off

pytestmark = pytest.mark.gpu
LARGE = 6.0e4


def make(B, Hq, Hk, Tq, Tk, D, dev, dt=torch.float16, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, H, T, D, generator=g) for H, T in ((Hq, Tq), (Hk, Tk), (Hk, Tk), (Hq, Tq)))
    return [t.to(dev, dt) for t in (q, k + 0.3, v + 0.5, 0.1 * do)]


def run(q, k, v, do, **kw):
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = ress.block_attention(*leaves, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, do)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk", [(256, 320), (700, 1374), (130, 9000)])
def test_large_values_in_dropped_blocks(dev, dt, D, Tq, Tk):
    """Key blocks that no row keeps, and rows that keep none: the same bits whatever finite values they hold."""
    q, k, v, do = make(1, 4, 2, Tq, Tk, D, dev, dt)
    g = torch.Generator().manual_seed(1)
    nq, nk = -(-Tq // 128), -(-Tk // 64)
    m = torch.rand(1, 4, nq, nk, generator=g) < 0.5
    m[..., 0] = True
    m[..., 1] = m[..., nk - 1] = False
    m[:, :, nq - 1] = False
    m = m.to(dev)
    want = run(q, k, v, do, block_map=m)
    for t in (k, v):
        t[:, :, 64:128] = LARGE
        t[:, :, (nk - 1) * 64:] = -LARGE
    q[:, :, (nq - 1) * 128:] = LARGE
    do[:, :, (nq - 1) * 128:] = LARGE
    got = run(q, k, v, do, block_map=m)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk,T", [(2, 2, 300), (4, 2, 700), (1, 1, 1500), (40, 40, 1340)])
def test_large_values_above_the_diagonal(dev, D, Hq, Hk, T):
    """Causal: values of the last 20 tokens reach no row before them, and their rows' gradients of the first 20 no key behind them."""
    q, k, v, do = make(1, Hq, Hk, T, T, D, dev)
    want = run(q, k, v, do, causal=True)
    late = v.clone()
    late[:, :, T - 20:] = LARGE
    got = run(q, k, late, do, causal=True)
    for i in (0, 1):
        assert torch.equal(got[i][:, :, :T - 20], want[i][:, :, :T - 20])
    early = do.clone()
    early[:, :, :20] = LARGE
    got = run(q, k, v, early, causal=True)
    for i in (2, 3):
        assert torch.equal(got[i][:, :, 20:], want[i][:, :, 20:])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk", [(200, 1374), (1374, 1374), (60, 21000)])
def test_one_large_value(dev, D, Tq, Tk):
    """A row's gradient that is 10^5 times the others', and a value of 6e4 that weighs nothing for the others, leave the others' dQ and dK at the error
    of the same roundings (norms over 59 rows or more: less than half apart)."""
    q, k, v, do = make(1, 1, 1, Tq, Tk, D, dev)
    q[..., 0] = 1.5
    k[:, :, 7] = 0.0
    k[:, :, 7, 0] = -200.0
    v[:, :, 7] = LARGE
    do[:, :, 3] *= 1.0e5
    q[:, :, 3], q[:, :, 3, 0] = 0.0, -20.0  # the row sees key 7 alone
    see = visible(1, 1, Tq, Tk)
    got, exact, like = run(q, k, v, do), attention(q, k, v, see, do), attention(q, k, v, see, do, torch.float16)
    rows = [i for i in range(Tq) if i != 3]
    keys = [j for j in range(Tk) if j != 7]
    for n, at in ((1, rows), (2, keys)):
        floor = 2.0 ** -25 * len(at) ** 0.5 * D ** 0.5 / exact[n][:, :, at].norm().item()  # fp16's smallest step
        assert off(got[n][:, :, at], exact[n][:, :, at]) <= 1.5 * off(like[n][:, :, at], exact[n][:, :, at]) + floor


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("H,Tq,Tk", [(1, 130, 3000), (3, 1500, 70), (2, 900, 900)])
def test_gradients_of_every_size(dev, D, rising, H, Tq, Tk):
    """Rows' gradients and keys' values of sizes from 2^-16 to 2^12 along the axes, up or down: dQ, each row by its own size, and dK in groups of
    32 at the error of the same roundings. The largest few rows make most of dK's error, so that the norms of two independent ones
    may differ by more than half: three times, and 2^-14 of the values for sums in 32 bits."""
    q, k, v, do = make(1, H, H, Tq, Tk, D, dev)
    size = [2.0 ** (28 * torch.arange(T, device=dev) / T - 16) for T in (Tq, Tk)]
    if not rising:
        size = [x.flip(0) for x in size]
    do = (do * size[0][:, None]).half()
    v = ((v - 0.5) * size[1][:, None]).half()
    see = visible(1, 1, Tq, Tk)
    got, exact, like = run(q, k, v, do), attention(q, k, v, see, do), attention(q, k, v, see, do, torch.float16)
    for n, unit in ((1, size[0][:, None].double()), (2, 1.0)):
        held = exact[n].abs() < 6.0e4  # by fp16: its largest number is 65,504
        error, same = (torch.where(held, t.double() - exact[n], 0.0) / unit for t in (got[n], like[n]))
        floor = torch.full_like(exact[n], 2.0 ** -25) / unit
        for x, y, z, f in zip(*(t.split(32, 2) for t in (error, same, exact[n] / unit, floor))):
            assert x.norm() <= 3.0 * y.norm() + 2.0 ** -14 * z.norm() + f.norm()
