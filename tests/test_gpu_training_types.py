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
