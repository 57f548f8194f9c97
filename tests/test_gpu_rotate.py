"""ress_amd.rotate and its gradients against the definition in 64 bits. Tolerances: half a step of the result's type, and 2^-22 of the
products' magnitudes (cosines and sines rounded to 32 bits, a product and a multiply-add)."""

import math

import pytest
import torch

import ress_amd as ress

pytestmark = pytest.mark.gpu
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def angles(rope, pos, base, d, scaling=None):
    inv = base ** (-torch.arange(0, d, 2, dtype=torch.float64, device=pos.device) / d)
    return pos.double()[..., None] * inv


def turned(x, pos, layout, axes, dims, base, sign=1.0):
    """(value, sum of magnitudes) of x (B, H, n, D) turned, pos (B, n, axes), as complex numbers."""
    d = dims // axes
    x = x.detach().double()
    inv = base ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    y, mag = x.clone(), torch.zeros_like(x)
    for a in range(axes):
        at = torch.arange(a * d, a * d + d, device=x.device)
        i1, i2 = (at[: d // 2], at[d // 2:]) if layout == "half" else (at[0::2], at[1::2])
        z = torch.complex(x[..., i1], x[..., i2])
        ang = sign * pos[..., a].double()[:, None, :, None] * inv
        z = z * torch.polar(torch.ones_like(ang), ang)
        y[..., i1], y[..., i2] = z.real, z.imag
        mag[..., i1] = mag[..., i2] = x[..., i1].abs() + x[..., i2].abs()
    return y, mag


def near(got, want, mag):
    bound = STEP[got.dtype] * want.abs() + 2.0 ** -22 * mag + (2.0 ** -25 if got.dtype is torch.float16 else 0.0)
    assert got.shape == want.shape and ((got.double() - want).abs() <= bound).all()


def make(B, H, n, D, dt, seed=0, layout="heads"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, n, D, generator=g).to(dt).cuda()
    if layout == "tokens":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "odd":
        x = torch.zeros(B, H, n, D + 3, dtype=dt, device="cuda")[..., 3:].copy_(x)
    return x.requires_grad_()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,axes,dims", [(64, 1, 64), (128, 1, 128), (64, 2, 64), (128, 2, 128), (128, 1, 64), (64, 2, 32), (64, 1, 24), (64, 2, 44),
                                         (64, 1, 2), (128, 1, 98), (64, 2, 4)])
@pytest.mark.parametrize("where", ["heads", "tokens", "odd"])
def test_layouts(dev, dt, layout, D, axes, dims, where):
    base = 1000.0
    q, k = make(2, 5, 37, D, dt, 1, where), make(2, 2, 37, D, dt, 2, where)
    rope = ress.RotaryTable(D, 300, base=base, axes=axes, device=dev, layout=layout, rotary_dim=dims)
    pos = torch.randint(0, 300, (2, 37, axes), generator=torch.Generator().manual_seed(3)).to(dev)
    given = pos[..., 0] if axes == 1 else pos
    outs = ress.rotate((q, k), given, rope)
    dy = [torch.randn(t.shape, generator=torch.Generator().manual_seed(4)).to(dev, dt) for t in (q, k)]
    grads = torch.autograd.grad(outs, (q, k), dy)
    for x, y, g, dx in zip((q, k), outs, dy, grads):
        near(y, *turned(x, pos, layout, axes, dims, base))
        near(dx, *turned(g, pos, layout, axes, dims, base, -1.0))
    with torch.no_grad():
        one = ress.rotate(q, given.to(torch.int32), rope)
        assert torch.equal(one, outs[0])
        assert torch.equal(ress.rotate(q[:1], given[0], rope), outs[0][:1])
    rope.check()


@pytest.mark.parametrize("B,H,n", [(1, 1, 1), (32, 40, 1), (1, 2, 5000), (3, 16, 1374), (2, 300, 3)])
def test_sizes(dev, B, H, n):
    x = make(B, H, n, 64, torch.bfloat16)
    rope = ress.RotaryTable(64, 6000, base=10000.0, axes=1, device=dev)
    pos = (torch.arange(n, device=dev)[None] + torch.arange(B, device=dev)[:, None] * 7) % 6000
    near(ress.rotate(x, pos, rope), *turned(x, pos[..., None], "half", 1, 64, 10000.0))


def test_far_positions(dev):
    """Angles of positions near a million are formed in 64 bits."""
    rope = ress.RotaryTable(64, 1_000_000, base=10000.0, axes=1, device=dev, layout="interleaved")
    x = make(1, 2, 50, 64, torch.float16)
    pos = 999_999 - torch.arange(50, device=dev)
    near(ress.rotate(x, pos, rope), *turned(x, pos[None, :, None], "interleaved", 1, 64, 10000.0))


def test_turned_keys_as_the_cache_turns_them(dev):
    """The same table, by halves: what PagedKVCache.append makes of queries, bit for bit but for the order of a sum."""
    from ress_amd import PagedKVCache, RotaryTable
    q, k = make(1, 4, 100, 64, torch.bfloat16).detach(), make(1, 2, 100, 64, torch.bfloat16, 1).detach()
    rope = RotaryTable(64, 128, axes=2, device=dev)
    pos = torch.randint(0, 128, (1, 100, 2), generator=torch.Generator().manual_seed(0)).to(dev)
    cache = PagedKVCache(4, 2, device=dev)
    got = cache.append(k, k, pos=pos, rope=rope, q=q)
    mine = ress.rotate(q, pos, rope)
    _, mag = turned(q, pos, "half", 2, 64, 100.0)
    assert ((got.double() - mine.double()).abs() <= 2 * STEP[q.dtype] * mine.double().abs() + 2.0 ** -21 * mag).all()


def test_a_position_outside_the_table(dev):
    rope = ress.RotaryTable(64, 10, axes=1, device=dev)
    x = make(1, 1, 3, 64, torch.bfloat16).detach()
    got = ress.rotate(x, torch.tensor([-5, 3, 99], device=dev), rope)
    assert torch.equal(got, ress.rotate(x, torch.tensor([0, 3, 9], device=dev), rope))
    with pytest.raises(RuntimeError, match="outside the rotation table"):
        rope.check()
    rope.check()


def test_gradients_of_one_operand_and_of_shared_positions(dev):
    q, k = make(2, 4, 10, 64, torch.bfloat16), make(2, 2, 10, 64, torch.bfloat16, 1)
    rope = ress.RotaryTable(64, 64, axes=1, device=dev)
    pos = torch.arange(10, device=dev)
    yq, yk = ress.rotate((q, k), pos, rope)
    g = torch.randn_like(k)
    a, = torch.autograd.grad(yk, k, g)
    b, = torch.autograd.grad(ress.rotate(k, pos, rope), k, g)
    assert torch.equal(a, b)
    x = q[:1, :1].detach().requires_grad_()
    y = ress.rotate(x.expand(2, 4, -1, -1), pos, rope)
    g = torch.ones_like(y)
    got, = torch.autograd.grad(y, x, g)
    full, = torch.autograd.grad(ress.rotate(q, pos, rope), q, g)
    assert torch.equal(got, full.sum((0, 1), keepdim=True))


def test_empty(dev):
    rope = ress.RotaryTable(64, 64, axes=1, device=dev)
    for B, H, n in ((0, 2, 3), (2, 0, 3), (2, 2, 0)):
        x = torch.zeros(B, H, n, 64, dtype=torch.float16, device=dev, requires_grad=True)
        y = ress.rotate(x, torch.zeros(B, n, dtype=torch.int64, device=dev), rope)
        assert torch.autograd.grad(y, x, torch.zeros_like(y))[0].shape == x.shape


def test_captured(dev):
    q, k = make(1, 4, 20, 64, torch.bfloat16), make(1, 2, 20, 64, torch.bfloat16, 1)
    rope = ress.RotaryTable(64, 512, axes=1, device=dev)
    pos = torch.arange(20, device=dev)
    g = [torch.randn_like(t) for t in (q, k)]

    def run(a, b, p):
        ys = ress.rotate((a, b), p, rope)
        return (*ys, *torch.autograd.grad(ys, (a, b), g))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(q, k, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(q, k, pos)
    for i in range(4):
        new = make(1, 4, 20, 64, torch.bfloat16, 10 + i), make(1, 2, 20, 64, torch.bfloat16, 20 + i)
        with torch.no_grad():
            q.copy_(new[0])
            k.copy_(new[1])
            pos.copy_(torch.arange(20, device=dev) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = run(*new, pos.clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 16.0, "original": 2048}])
def test_scaled_tables(dev, scaling):
    """The table's own rows, as it holds them (their values: test_rotary_tables.py)."""
    rope = ress.RotaryTable(64, 9000, base=10000.0, axes=1, device=dev, scaling=scaling)
    x = make(1, 1, 4, 64, torch.bfloat16)
    pos = torch.tensor([0, 1, 4000, 8999], device=dev)
    c, s = rope.table[pos].double().unbind(1)
    v = x.detach().double()[0, 0]
    want = torch.cat([v[:, :32] * c - v[:, 32:] * s, v[:, 32:] * c + v[:, :32] * s], -1)[None, None]
    mag = (v.abs() + v.roll(32, -1).abs())[None, None] * math.sqrt(2)
    near(ress.rotate(x, pos, rope), want, mag)


def test_offsets_past_32_bits(dev):
    """More than 2^32 elements, there and back: the last tokens as a call of their own."""
    n, few = (1 << 24) + 37, 100
    x = torch.randn(1, 2, few, 128, generator=torch.Generator().manual_seed(0)).to(dev, torch.bfloat16)
    rope = ress.RotaryTable(128, few, base=1000.0, axes=1, device=dev, layout="interleaved")
    pos = torch.arange(n, device=dev) % few
    many = x.repeat(1, 1, -(-n // few), 1)[:, :, :n].contiguous().requires_grad_()
    y = ress.rotate(many, pos, rope)
    want = ress.rotate(x, pos[:few], rope)
    last = n // few * few
    assert torch.equal(y[:, :, :few], want) and torch.equal(y[:, :, last:], want[:, :, :n - last])
    back, = torch.autograd.grad(y, many, y.detach())
    again = ress.rotate(x.requires_grad_(), pos[:few], rope)
    want, = torch.autograd.grad(again, x, again.detach())
    assert torch.equal(back[:, :, :few], want) and torch.equal(back[:, :, last:], want[:, :, :n - last])
