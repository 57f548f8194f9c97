"""The linear layer in 8-bit integers: codes, products and the layer, against 64 bits."""

import math

import pytest
import torch
import torch.nn as nn

from ress_amd.int8 import Int8Linear, int8_linear, quantize_linears, quantize_tokens, quantize_weight

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _rand(shape, dtype, dev, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * gain).to(dtype).to(dev)


def _weights(N, K, dev, seed, bias=True):
    codes, scale = quantize_weight(_rand((N, K), torch.float32, dev, seed, K ** -0.5))
    return codes, scale, _rand((N,), torch.float32, dev, seed + 1, 0.3) if bias else None


def _expected(x, codes, scale, bias, act):
    """(y, allowed error): from the codes that quantize_tokens gives, in 64 bits. fp32: the sum's conversion, two
    products and an addition, half a step each of their results; erf and its products a few units more (2^-20);
    the output half a step of its type."""
    c, s = quantize_tokens(x)
    p = (c.double().cpu() @ codes.double().cpu().T) * s.double().cpu()[..., None] * scale.double().cpu()
    y = p if bias is None else p + bias.double().cpu()
    err = 3 * 2.0 ** -24 * p.abs() + 2.0 ** -24 * y.abs()
    if act == "gelu":
        err = 1.13 * err + 2.0 ** -20 * y.abs()
        y = y * torch.special.ndtr(y)
    u = torch.finfo(x.dtype).eps / 2
    return y, err * (1 + u) + u * y.abs() + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps


def _check(x, codes, scale, bias, act, got):
    want, tol = _expected(x, codes, scale, bias, act)
    err = (got.double().cpu() - want).abs()
    assert got.dtype == x.dtype and got.shape == want.shape
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("K", [16, 64, 1008, 4096, 6000])
def test_codes(dev, dtype, K):
    """Within half a step; the factor 127 / a and the product with it are off by 2 * 2^-24 of up to 127 steps."""
    for off in (0, 1):
        x = _rand((7 * K + 1,), dtype, dev, K)[off:off + 7 * K].view(7, K)
        x = x * torch.tensor([1, 1e-3, 30, 0, 1, 1, 1], device=dev).to(dtype)[:, None] if off == 0 else x
        c, s = quantize_tokens(x)
        xd = x.double().cpu()
        top = xd.abs().amax(1)
        assert ((s.double().cpu() - top / 127).abs() <= top / 127 * 2.0 ** -22).all()
        assert ((c.double().cpu() * s.double().cpu()[:, None] - xd).abs() <= (top / 127)[:, None] * (0.5 + 127 * 2.0 ** -21)).all()
        assert (c.abs().amax(1).cpu() == torch.where(top > 0, 127, 0)).all()
    # the smallest magnitudes of the type
    tiny = torch.zeros(2, K, dtype=dtype, device=dev)
    tiny[0, 3] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    c, s = quantize_tokens(tiny)
    assert ((c.float() * s[:, None] - tiny.float()).abs() <= tiny.float().amax()).all() and (c[1] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M", [1, 2, 9, 16, 17, 127, 130, 300])
@pytest.mark.parametrize("K,N", [(16, 5), (48, 130), (128, 128), (144, 3), (1024, 260), (1040, 1024), (4112, 520), (2560, 2080)])
def test_products(dev, dtype, M, K, N):
    codes, scale, bias = _weights(N, K, dev, K)
    x = _rand((M, K), dtype, dev, M)
    for b, act in ((bias, None), (None, "gelu")):
        _check(x, codes, scale, b, act, int8_linear(x, codes, scale, b, act))


def test_large_sums(dev):
    """Every code at its largest: the sum passes 2^24 and stays exact in int32."""
    K = 131072
    x = torch.ones(3, K, dtype=BF16, device=dev)
    codes, scale = torch.full((4, K), 127, dtype=torch.int8, device=dev), torch.ones(4, device=dev) / 127
    got = int8_linear(x, codes, scale)
    _check(x, codes, scale, None, None, got)
    x = torch.ones(20, K, dtype=BF16, device=dev)
    _check(x, codes, scale, None, None, int8_linear(x, codes, scale))


@pytest.mark.parametrize("M", [3, 40])
def test_largest_activations(dev, M):
    """Near bf16's end: the sum times a token's scale would pass it, times both scales it does not."""
    codes, scale, bias = _weights(36, 1024, dev, 5)
    x = _rand((M, 1024), BF16, dev, 6, 2.0 ** 120)
    _check(x, codes, scale, bias, None, int8_linear(x, codes, scale, bias))


@pytest.mark.parametrize("M", [3, 40])
def test_layouts(dev, M):
    """Leading dims, rows of a wider tensor, odd offsets: as a copy does."""
    K, N = 96, 70
    codes, scale, bias = _weights(N, K, dev, 1)
    x = _rand((2, M, K), BF16, dev, 2)
    want = int8_linear(x, codes, scale, bias)
    _check(x, codes, scale, bias, None, want)
    wide = torch.zeros(2 * M, K + 8, dtype=BF16, device=dev)
    wide[:, :K] = x.view(-1, K)
    odd = torch.zeros(2 * M * K + 1, dtype=BF16, device=dev)
    odd[1:] = x.flatten()
    for y in (wide[:, :K], odd[1:].view(2, M, K), x.transpose(0, 1).contiguous().transpose(0, 1), x[:1].expand(2, M, K)):
        got = int8_linear(y, codes, scale, bias)
        ref = int8_linear(y.contiguous(), codes, scale, bias)
        assert torch.equal(got, ref)
    assert torch.equal(int8_linear(wide[:, :K], codes, scale, bias), want.view(-1, N))
    assert torch.equal(int8_linear(x[0, 0], codes, scale, bias), want[0, 0])
    assert int8_linear(x[:, :0], codes, scale).shape == (2, 0, N)


@pytest.mark.parametrize("M", [4, 50])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_that_are_not_finite(dev, dtype, M):
    codes, scale, bias = _weights(40, 64, dev, 1)
    x = _rand((M, 64), dtype, dev, 2)
    want = int8_linear(x, codes, scale, bias)
    for bad in (math.nan, math.inf, -math.inf):
        y = x.clone()
        y[2, 5] = bad
        got = int8_linear(y, codes, scale, bias)
        assert got[2].isnan().all()
        got[2] = want[2]
        assert torch.equal(got, want)
        c, s = quantize_tokens(y)
        assert s[2].isnan() and (c[2] == 0).all()


def test_weight(dev):
    w = _rand((33, 64), torch.float32, dev, 3)
    w[4] = 0
    c, s = quantize_weight(w)
    step = w.double().abs().amax(1) / 127
    assert ((c.double() * s.double()[:, None] - w.double()).abs() <= step[:, None] * (0.5 + 127 * 2.0 ** -21)).all()
    assert s[4] == 0 and (c[4] == 0).all()
    w[2, 2] = math.inf
    with pytest.raises(ValueError, match="not finite"):
        quantize_weight(w)


def test_layer_and_model(dev):
    torch.manual_seed(0)
    layer = nn.Linear(64, 48).to(dev, BF16)
    q = Int8Linear(layer)
    x = _rand((5, 64), BF16, dev, 1)
    with torch.no_grad():
        assert torch.equal(q(x), int8_linear(x, *quantize_weight(layer.weight), layer.bias.float()))
        assert (q.weight.float() - layer.weight.float()).abs().max() <= layer.weight.abs().max().float() / 127
    assert q.weight.dtype == BF16
    s = q.scale.clone()
    assert torch.equal(q.to(F16).scale, s) and q.bias.dtype == torch.float32 and q.codes.dtype == torch.int8
    model = nn.Sequential(nn.Linear(64, 32), nn.GELU(), nn.Sequential(nn.Linear(32, 20), nn.Linear(20, 8))).to(dev, BF16)
    names = quantize_linears(model, keep=lambda name, linear: name == "2.0")
    assert names == ["0"] and type(model[2][0]) is nn.Linear and type(model[2][1]) is nn.Linear
    with torch.no_grad():
        assert model(x).shape == (5, 8)


@pytest.mark.parametrize("M", [2, 60])
def test_captured(dev, M):
    codes, scale, bias = _weights(200, 256, dev, 1)
    x = _rand((M, 256), BF16, dev, 2)
    int8_linear(x, codes, scale, bias, "gelu")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = int8_linear(x, codes, scale, bias, "gelu")
    for seed in range(3):
        x.copy_(_rand((M, 256), BF16, dev, 10 + seed))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, int8_linear(x, codes, scale, bias, "gelu"))


def test_refusals(dev):
    codes, scale, bias = _weights(8, 32, dev, 1)
    x = _rand((4, 32), BF16, dev, 2)
    for bad, err in ((x.cpu(), RuntimeError), (x.float(), TypeError), (x[:, :24], ValueError), (x[:, :0], ValueError),
                     (x[:, :16], ValueError)):
        with pytest.raises(err):
            int8_linear(bad, codes, scale)
    with pytest.raises(ValueError, match="w_codes"):
        int8_linear(x, codes.float(), scale)
    with pytest.raises(ValueError, match="w_codes"):
        int8_linear(x, codes.repeat(1, 2)[:, ::2], scale)
    with pytest.raises(ValueError, match="w_scale"):
        int8_linear(x, codes, scale.half())
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, codes, scale, bias[:4])
    with pytest.raises(ValueError, match="are not on"):
        int8_linear(x, codes, scale.cpu())
    with pytest.raises(ValueError, match="act"):
        int8_linear(x, codes, scale, act="relu")
    with pytest.raises(RuntimeError, match="no backward"):
        int8_linear(x.clone().requires_grad_(), codes, scale)
    with pytest.raises(RuntimeError, match="device tensor"):
        quantize_tokens(x.cpu())
    with pytest.raises(ValueError, match="rows"):
        quantize_tokens(x[:1].expand((1 << 30) + 1, 32))
