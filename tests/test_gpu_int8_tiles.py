"""Every tile that the 8-bit product is cut into, with K a multiple of 256 and not, against 64 bits."""

import pytest
import torch

from ress_amd import _lib
from ress_amd.int8 import int8_linear, quantize_tokens

# (tokens, channels of a tile): products that take it, M and N no multiples of it
SHAPES = {
    (256, 256): [(3000, 1024, 4090), (3000, 1040, 4090), (6000, 272, 2052)],
    (192, 256): [(2050, 1024, 4090), (8200, 1024, 1032), (8200, 272, 1000), (4097, 272, 2052)],
    (128, 128): [(1374, 1024, 4090), (2050, 1024, 3000), (4097, 1040, 1000), (2050, 272, 3000)],
    (64, 128): [(3000, 1024, 1000), (1374, 1024, 2052), (3000, 272, 1032), (3000, 272, 1002)],
    (64, 64): [(300, 1024, 250), (700, 1024, 1000), (300, 1040, 250), (700, 272, 252), (17, 4112, 1030)],
}
CASES = [(tile, *s) for tile, shapes in SHAPES.items() for s in shapes]


@pytest.mark.parametrize("tile,M,K,N", CASES)
def test_tile_of_a_product(tile, M, K, N):
    got = _lib.lib().ress_int8_linear_tile(M, K, N)
    assert (got >> 16, got & 0xffff) == tile


def test_every_tile_is_met():
    for tile, shapes in SHAPES.items():
        assert {K % 256 == 0 for _, K, _ in shapes} == {True, False}
        assert {N % 4 == 0 for _, _, N in shapes} == {True, False}
    assert _lib.lib().ress_int8_linear_tile(16, 1024, 4096) == _lib.lib().ress_int8_linear_tile(0, 16, 16) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tile,M,K,N", CASES)
def test_products(dev, dtype, tile, M, K, N):
    """The sum of the codes' products in 64 bits is exact. fp32: its conversion, two products and an addition, half a step
    (2^-24) each of their results; gelu, of slope 1.13 at most, by an approximation within 2^-22 of its argument and a few
    units of 2^-24 (2^-20 in all); the output half a step of its type."""
    g = torch.Generator().manual_seed(M + K + N)
    x = (torch.randn(M, K, generator=g) * torch.rand(M, 1, generator=g)).to(dev, dtype)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).to(dev)
    scale = ((torch.rand(N, generator=g) + 0.5) * K ** -0.5 / 127).to(dev)
    bias = torch.randn(N, generator=g).to(dev)
    c, s = quantize_tokens(x)
    p = (c.double() @ w.double().t().contiguous()) * s.double()[:, None] * scale.double()
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for b, act in ((bias, None), (None, "gelu")):
        y = p if b is None else p + b.double()
        err = 3 * 2.0 ** -24 * p.abs() + 2.0 ** -24 * y.abs()
        if act == "gelu":
            err = 1.13 * err + 2.0 ** -20 * y.abs()
            y = y * torch.special.ndtr(y)
        got = int8_linear(x, w, scale, b, act)
        assert got.shape == (M, N) and got.dtype == dtype
        off = (got.double() - y).abs()
        assert (off <= err * (1 + u) + u * y.abs() + tiny).all(), (act, float((off / (u * y.abs() + tiny)).max()))
