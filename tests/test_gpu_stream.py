"""Frames streamed through a model over 8-bit caches: append and attention as a layer calls them, the model's
steps, and its layers in 8-bit integers."""

import math

import pytest
import torch
import torch.nn.functional as F

from kvcache_oracle import PAGE, attention, half_step, held, tolerance
from ress_amd import FrameStream, quantize_linears
from ress_amd.aggregator import Attention, Mlp, RoPE2D, build_vggt_aggregator, synthetic_frames
from ress_amd.int8 import Int8Linear
from ress_amd.kvcache import PagedKVCache
from ress_amd.qkv import fused_qk_norm_rope
from ress_amd.stream import cached_attention

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _attn(dev, dtype, dim, heads, seed=0):
    torch.manual_seed(seed)
    a = Attention(dim, heads, RoPE2D()).to(dev, dtype).eval()
    a.proj = torch.nn.Identity()
    return a


def _tokens(dev, dtype, B, T, dim, seed=1):
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, 38, (B, T, 2), generator=g).to(dev)
    return torch.randn(B, T, dim, generator=g).to(dev, dtype), pos


@pytest.mark.parametrize("dtype,dim,heads", [(BF16, 128, 2), (F16, 128, 2), (BF16, 256, 2), (F16, 256, 2)])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_layer_over_cache(dev, dtype, dim, heads, codes):
    """Three calls of a layer (the fused norms and rotation in bf16 with head dim 64, else the rotation of append)
    against attention in 64 bits over what the cache holds."""
    attn = _attn(dev, dtype, dim, heads)
    c = PagedKVCache(20, heads, dim // heads, max_seqs=2, max_len=400, dtype=dtype, codes=codes, device=dev)
    B = 2
    with torch.no_grad():
        for T in (70, 1, 137):
            x, pos = _tokens(dev, dtype, B, T, dim, seed=T)
            got = cached_attention(attn, x, pos, c, {})
            if dtype == BF16 and dim // heads == 64:
                q = fused_qk_norm_rope(attn, attn.qkv(x), pos, heads)[0]
            else:
                q = attn.rope(attn.q_norm(attn.qkv(x).reshape(B, T, 3, heads, -1)[:, :, 0].transpose(1, 2)), pos)
            for b in range(B):
                k, v = held(c, b)
                want, size, spread = attention(q[b], k, v, T, False)
                tol = tolerance(want, size, spread, dtype, k.shape[1])
                # the module's rotation and append's round the same query apart by up to one step in rare places
                tol = tol + (size + want.abs()) * 4 * half_step(dtype) * spread if dtype == F16 or dim // heads != 64 else tol
                err = (got[b].reshape(T, heads, -1).transpose(0, 1).double().cpu() - want).abs()
                assert (err <= tol).all(), float((err / tol).max())
    c.check()


def test_quantisation_error_of_a_layer(dev):
    """Against the same layer's dense attention in fp32 over unquantised keys and values: each key is off by at most
    half a code step a dim, which moves a score by at most d = scale * sum |q| * step / 2 and a weight by a factor
    within e^(+-2 d); each value by half a step. 16-bit P and output: half a step each."""
    dim, heads, T = 128, 2, 500
    attn = _attn(dev, BF16, dim, heads)
    x, pos = _tokens(dev, BF16, 1, T, dim)
    c = PagedKVCache(10, heads, 64, max_len=T, device=dev)
    with torch.no_grad():
        got = cached_attention(attn, x, pos, c, {}).reshape(T, heads, 64).transpose(0, 1).double().cpu()
        q, k, v = (t[0].double().cpu() for t in fused_qk_norm_rope(attn, attn.qkv(x), pos, heads))
    p = torch.softmax(q @ k.transpose(1, 2) / 8, -1)
    want, size = p @ v, p @ v.abs()
    ids = c.table[0, :T // PAGE].long().cpu()
    step_k, step_v = (s.cpu().double()[ids].amax(0)[:, None, None] * (0.5 + 2.0 ** -14) for s in (c.k_scale, c.v_scale))
    d = q.abs().sum(-1, keepdim=True) / 8 * step_k
    tol = torch.expm1(2 * d) * (size + step_v) + step_v + 2 * half_step(BF16) * (size + want.abs())
    assert ((got - want).abs() <= tol).all()
    assert (got - want).norm() / want.norm() < 0.02  # half a step of 127 beside values of 1/3 to 1/4 of the largest


def _model(dev, dtype=BF16, depth=2):
    return build_vggt_aggregator(depth=depth, dim=128, num_heads=2, device=dev, dtype=dtype)


@pytest.mark.parametrize("dtype,codes", [(BF16, "int8"), (F16, "fp8")])
def test_stream_of_frames(dev, dtype, codes):
    model = _model(dev, dtype)
    frames = synthetic_frames(4, size=112, B=2, device=dev)
    P = 8 * 8 + 5
    s = FrameStream(model, 4, batch=2, codes=codes)
    first = s.step(frames[:, 0])
    assert first.shape == (2, P, 128) and first.dtype == dtype and torch.isfinite(first).all()
    snap = s.snapshot()
    second = s.step(frames[:, 1])
    s.step(frames[:, 2:4])
    assert s.frames == 4 and all(c.lengths() == [4 * P, 4 * P] for c in s.caches)
    with pytest.raises(ValueError, match="do not fit"):
        s.step(frames[:, :1])
    s.restore(snap)
    assert s.frames == 1 and torch.equal(s.step(frames[:, 1]), second)
    with pytest.raises(ValueError, match="patch grid"):
        s.step(synthetic_frames(1, size=126, B=2, device=dev))
    s.check()
    s.reset()
    assert s.frames == 0 and torch.equal(s.step(frames[:, 0]), first)
    s.reset()
    larger = synthetic_frames(4, size=126, B=2, device=dev)
    got = s.step(larger)
    assert s.frames == 4 and torch.equal(got, FrameStream(model, 4, batch=2, codes=codes).step(larger))
    s.check()
    s.reset()
    with pytest.raises(RuntimeError, match="graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            s.step(frames[:, 0])


def test_all_frames_in_one_step_is_the_dense_aggregator(dev):
    """What differs is the attention's quantisation (test_quantisation_error_of_a_layer: under 2% of its output) and
    the rounding of P, behind LayerScale 0.01 of a residual stream: under 2% of 0.01 of each of two layers, and what
    the 16-bit residual additions round apart (half a step of 2^-8 each, 4 a pair of blocks)."""
    model = _model(dev)
    dense = build_vggt_aggregator(depth=2, dim=128, num_heads=2, device=dev, wire=False)
    frames = synthetic_frames(3, size=112, device=dev)
    with torch.no_grad():
        want = dense.aggregator(frames).double()
        got = FrameStream(model, 3).step(frames).double()
    assert ((got - want).norm() / want.norm()).item() < 2 * 0.02 * 0.01 + 8 * half_step(BF16)
    # an error in the order of frames, positions or special tokens is not behind a factor of 0.01
    other = FrameStream(model, 3).step(frames.flip(1)).double()
    assert ((other - want).norm() / want.norm()).item() > 10 * ((got - want).norm() / want.norm()).item()


def test_stream_with_8_bit_layers(dev):
    model = _model(dev)
    names = quantize_linears(model)
    assert len(names) == 4 * 4 and all(n.endswith(("qkv", "proj", "fc1", "fc2")) for n in names)
    frames = synthetic_frames(2, size=112, device=dev)
    s = FrameStream(model, 2)
    for i in range(2):
        assert torch.isfinite(s.step(frames[:, i])).all()
    s.check()


def test_mlp_fuses_gelu(dev):
    """fc1 with its gelu fused rounds once where the modules round twice: by gelu's slope (at most 1.13) of half a
    step of its input, and half a step of the result, apart."""
    torch.manual_seed(0)
    m = Mlp(64, 256).to(dev, BF16)
    m.fc1 = Int8Linear(m.fc1)
    m.fc2 = torch.nn.Identity()
    x = torch.randn(50, 64, device=dev).to(BF16)
    with torch.no_grad():
        got, y = m(x).double(), m.fc1(x).double()
    want = F.gelu(y)
    u = half_step(BF16)
    assert ((got - want).abs() <= 1.13 * u * y.abs() * (1 + u) + u * (want.abs() + 1.13 * u * y.abs()) + 1e-6).all()


def test_a_step_that_fails_is_not_continued(dev):
    model = _model(dev)
    s = FrameStream(model, 3)
    frames = synthetic_frames(1, size=112, device=dev)
    s.step(frames)
    snap = s.snapshot()
    proj = model.aggregator.global_blocks[1].attn.proj
    model.aggregator.global_blocks[1].attn.proj = torch.nn.Linear(7, 7).to(dev, BF16)
    with pytest.raises(RuntimeError):
        s.step(frames)
    model.aggregator.global_blocks[1].attn.proj = proj
    with pytest.raises(RuntimeError, match="ended in an error"):
        s.step(frames)
    s.restore(snap)
    s.step(frames)
    assert s.frames == 2 and math.isfinite(s.step(frames).float().sum().item())
