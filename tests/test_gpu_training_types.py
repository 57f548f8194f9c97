"""The types that wired layers compute and record in with gradients."""

import math

import pytest
import torch

import ress_amd as ress
from ress_amd import training
from ress_amd.aggregator import build_vggt_aggregator, synthetic_frames
from ress_amd.wiring import wire_ress_attention

pytestmark = pytest.mark.gpu


def wired(dtype, mode, record=False):
    model = build_vggt_aggregator(depth=1, dim=128, num_heads=2, seed=0, dtype=torch.float32).to(dtype)
    stores = [{}] if record else None
    if record:
        wire_ress_attention(model, model.aggregator.global_blocks, stores)
    if mode == "dense":
        model.aggregator.global_blocks[0].attn.dense = True
    else:
        ress.apply_sparse_vggt(model, sparse_ratio=0.5)
    return ress.enable_gradients(model), stores


def layer(model, dtype, dev):
    """(attention, x, pos) of the model's wired layer, over two frames of 12 x 12 patches and 5 special tokens."""
    attn = model.aggregator.global_blocks[0].attn
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 2 * 149, 128, generator=g).to(dev, dtype)
    i = torch.arange(149) - 5
    pos = torch.stack([torch.where(i < 0, 0, i // 12 + 1), torch.where(i < 0, 0, i % 12 + 1)], -1).repeat(2, 1)[None].to(dev)
    return attn, x, pos


@pytest.mark.parametrize("mode", ["sparse_vggt", "dense"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_models_compute_in_their_type(dev, monkeypatch, mode, dtype):
    model, _ = wired(dtype, mode)
    attn, x, pos = layer(model, dtype, dev)
    seen, block_attention = [], training.block_attention
    monkeypatch.setattr(training, "block_attention", lambda q, k, v, **kw: (seen.append({t.dtype for t in (q, k, v)}),
                                                                             block_attention(q, k, v, **kw))[1])
    attn(x, pos).float().sum().backward()
    assert seen == [{dtype}]


def test_a_dense_32_bit_layer_keeps_32_bits(dev):
    """As without the operators, and its gradients: sums of 32-bit products (2^-24 each, over up to 298 keys and 128 channels in a
    few steps, some of which cancel: 2^-14 of the largest value)."""
    model, _ = wired(torch.float32, "dense")
    attn, x, pos = layer(model, torch.float32, dev)
    x.requires_grad_()
    got = attn(x, pos)
    dx, = torch.autograd.grad(got, x, torch.ones_like(got))
    ress.enable_gradients(model, on=False)
    want = attn(x, pos)
    dw, = torch.autograd.grad(want, x, torch.ones_like(want))
    assert got.dtype == torch.float32
    assert (got - want).abs().max() <= 2.0 ** -14 * want.abs().max() and (dx - dw).abs().max() <= 2.0 ** -14 * dw.abs().max()


@pytest.mark.parametrize("mode", ["sparse_vggt", "dense"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_recorded_outputs_and_their_gradients_have_32_bits(dev, mode, dtype):
    """As without the operators: a head score is made of the gradient's square."""
    model, stores = wired(dtype, mode, record=True)
    attn, x, pos = layer(model, dtype, dev)
    attn.retain_output_grad = True
    out = attn(x, pos)
    assert out.dtype == dtype
    (out.float() * torch.linspace(-1, 1, out.numel(), device=dev).view_as(out)).sum().backward()
    o = stores[0]["value"].output
    assert o.dtype == torch.float32 and o.shape == (1, 2, 298, 64)
    assert o.grad.dtype == torch.float32 and torch.isfinite(o.grad).all() and o.grad.abs().max() > 0
    assert attn.qkv.weight.grad.abs().max() > 0
    with torch.no_grad():
        attn(x, pos)
    off = (stores[0]["value"].output - o).abs().max() / o.abs().max()
    assert off <= math.ldexp(1.0, -5)  # the inference path's 8-bit scores


def test_queries_and_keys_under_autocast(dev):
    """As torch's modules under autocast: from the projection's rounding to the attention's operands one more, where a rounding between
    norm and rotation would make two (2^-8 of an element each, and its partner's share in it)."""
    block = build_vggt_aggregator(depth=1, dim=128, num_heads=2, seed=0, dtype=torch.float32, wire=False).aggregator.frame_blocks[0]
    attn = block.attn
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for norm in (attn.q_norm, attn.k_norm):
            norm.weight.copy_(1 + 0.3 * torch.randn(64, generator=g))
            norm.bias.copy_(0.3 * torch.randn(64, generator=g))
    qkv = torch.randn(2, 150, 384, generator=g).to(dev, torch.bfloat16).requires_grad_()
    pos = torch.randint(0, 37, (2, 150, 2), generator=g).to(dev)
    dy = torch.randn(2, 2, 2, 150, 64, generator=g).to(dev, torch.bfloat16)
    with torch.autocast("cuda", torch.bfloat16):
        got = training.normed_and_turned(attn, qkv, pos, 2)
    assert all(t.dtype == torch.bfloat16 for t in got)
    grad, = torch.autograd.grad(got[:2], qkv, list(dy))
    exact = qkv.detach().double().requires_grad_()
    heads = exact.view(2, 150, 3, 2, 64).permute(2, 0, 3, 1, 4)
    want = []
    for t, norm in zip(heads, (attn.q_norm, attn.k_norm)):
        t = torch.nn.functional.layer_norm(t, (64,), norm.weight.double(), norm.bias.double(), norm.eps)
        turned = []
        for axis in (0, 1):
            inv = 100.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64, device=dev) / 32)
            z = torch.complex(t[..., 32 * axis:32 * axis + 16], t[..., 32 * axis + 16:32 * axis + 32])
            z = z * torch.polar(torch.ones_like(inv), pos[:, None, :, axis, None].double() * inv)
            turned += [z.real, z.imag]
        want.append(torch.cat(turned, -1))
    for x, y in zip(got, want):
        # half a step, and 2^-17 of the elements' size: angles of up to 37 in 32 bits (the module's), products and sums
        assert ((x.double() - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -17 * y.abs().amax()).all()
    wanted, = torch.autograd.grad(want, exact, list(dy.double()))
    # the projection's gradient is rounded once, and so is dy turned back where the module hands on 16 bits
    assert ((grad.double() - wanted).norm() / wanted.norm()) <= 2.0 ** -8
