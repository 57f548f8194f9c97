"""Which rotary modules a table stands for under enable_gradients."""

import pytest
import torch
import torch.nn as nn

import ress_amd as ress
from ress_amd import training
from ress_amd.aggregator import Block, RoPE2D

pytestmark = pytest.mark.gpu


class Mirrored(RoPE2D):
    def forward(self, tokens, positions):
        return super().forward(tokens, -positions)


class Own(nn.Module):
    """A backbone's own module of the same arithmetic."""

    def __init__(self):
        super().__init__()
        self.inner = RoPE2D()

    def forward(self, tokens, positions):
        return self.inner(tokens, positions)


def block(dev, rope):
    torch.manual_seed(0)
    b = Block(128, 2, 2.0, rope).to(dev, torch.bfloat16)
    return ress.enable_gradients(b)


def inputs(dev, n=40):
    g = torch.Generator().manual_seed(1)
    return (torch.randn(2, n, 128, generator=g).to(dev, torch.bfloat16), torch.randint(1, 9, (2, n, 2), generator=g).to(dev))


def tables(rope):
    return rope.__dict__.get("_ress_rotary_tables", {})


def test_hooks_are_run(dev):
    b, (x, pos) = block(dev, RoPE2D()), inputs(dev)
    b(x, pos)
    assert tables(b.attn.rope)
    seen = []
    handle = b.attn.rope.register_forward_hook(lambda m, a, out: seen.append(a[0].shape))
    b(x, pos)
    assert len(seen) == 2
    handle.remove()
    b(x, pos)
    assert len(seen) == 2
    b.attn.rope.forward = lambda t, p: (seen.append(t.shape), t)[1]
    b(x, pos)
    assert len(seen) == 4


def test_a_subclass_runs_its_own_forward(dev):
    b, (x, pos) = block(dev, Mirrored()), inputs(dev)
    got = b(x, pos)
    assert not tables(b.attn.rope)
    plain = block(dev, RoPE2D())
    assert not torch.equal(got, plain(x, pos))
    qkv = torch.randn(2, 40, 384, device=dev).bfloat16()
    q, k, _ = training.normed_and_turned(b.attn, qkv, pos, 2)
    heads = qkv.view(2, 40, 3, 2, 64).permute(2, 0, 3, 1, 4)
    for got, t, norm in ((q, heads[0], b.attn.q_norm), (k, heads[1], b.attn.k_norm)):
        assert torch.equal(got, b.attn.rope(training._norm(norm, t), pos).to(got.dtype))


def test_a_declared_module_has_a_table(dev):
    x, pos = inputs(dev)
    rope = Own()
    assert not tables(rope)
    b = block(dev, rope)
    b(x, pos)
    assert not tables(rope)
    ress.declare_rope(rope, rope.inner.base)
    b(x, pos)
    assert tables(rope)


@pytest.mark.parametrize("n,last", [(1505, 1500), (40, 1023), (2100, 2100)])
def test_grids_of_more_than_1024_rows(dev, n, last):
    """Positions up to the number of tokens are turned as the module does, and none is reported."""
    rope = RoPE2D()
    b = block(dev, rope)
    x = torch.randn(1, n, 384, generator=torch.Generator().manual_seed(3)).to(dev, torch.bfloat16)
    pos = torch.stack([torch.arange(n), torch.arange(n).flip(0)], -1).clamp(max=last)[None].to(dev)
    pos[0, -1] = last
    for i, (got, norm) in enumerate(zip(training.normed_and_turned(b.attn, x, pos, 2)[:2], (b.attn.q_norm, b.attn.k_norm))):
        t = training._norm(norm, x.view(1, n, 3, 2, 64)[:, :, i].transpose(1, 2)).double()
        inv = 100.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64, device=dev) / 32)
        want = []
        for axis in (0, 1):
            z = torch.complex(t[..., 32 * axis:32 * axis + 16], t[..., 32 * axis + 16:32 * axis + 32])
            z = z * torch.polar(torch.ones_like(inv), pos[0, :, axis, None].double() * inv)
            want += [z.real, z.imag]
        want = torch.cat(want, -1)
        # the result's rounding, 2^-24 of cosines and sines and two products of them
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -21 * t.abs().amax()).all()
    ress.check_layers(b)


def test_a_known_grid_sizes_the_table(dev):
    rope = RoPE2D()
    b = block(dev, rope)
    pos = torch.zeros(1, 3000, 2, dtype=torch.int64, device=dev)
    pos.ress_patch_grid = (37, 37)
    training.normed_and_turned(b.attn, torch.zeros(1, 3000, 384, dtype=torch.bfloat16, device=dev), pos, 2)
    assert [len(t.table) for t in tables(rope).values()] == [1024]
    first, = tables(rope).values()
    pos = torch.full((1, 2000, 2), 1999, device=dev)
    training.normed_and_turned(b.attn, torch.zeros(1, 2000, 384, dtype=torch.bfloat16, device=dev), pos, 2)
    assert sorted(len(t.table) for t in tables(rope).values()) == [1024, 2048]
    assert any(t is first for t in tables(rope).values())  # a graph may read it
    ress.check_layers(b)
