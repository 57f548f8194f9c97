"""A model with 8-bit layers on the framework's own paths: the sparse layers, autocast, and a stream of its frames."""

import pytest
import torch

import ress_amd
from ress_amd import FrameStream, quantize_linears
from ress_amd.aggregator import build_vggt_aggregator, synthetic_frames
from ress_amd.int8 import int8_linear

pytestmark = pytest.mark.gpu


def _relative(got, want):
    return ((got.double() - want.double()).norm() / want.double().norm()).item()


def test_sparse_layers(dev):
    """Codes are off by up to half a step of 1/127 of a row's largest value, some 1% of an activation or weight: behind
    LayerScale 0.01 a forward of four blocks moves by far less than 1%."""
    model = build_vggt_aggregator(depth=2, dim=128, num_heads=2, device=dev)
    frames = synthetic_frames(3, size=112, device=dev)
    ress_amd.apply_sparse_vggt(model, sparse_ratio=0.3)
    with torch.no_grad():
        want = model(frames)
        assert len(quantize_linears(model)) == 16
        got = model(frames)
    assert torch.isfinite(got).all() and 0 < _relative(got, want) < 0.01


def test_autocast(dev):
    """A 32-bit layer under autocast: what int8_linear gives for the cast input."""
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(64, 48), torch.nn.Linear(48, 32)).to(dev)
    x = torch.randn(70, 64, device=dev)
    quantize_linears(m)
    with torch.no_grad():
        with pytest.raises(TypeError, match="autocast"):
            m(x)
        for dtype in (torch.bfloat16, torch.float16):
            with torch.autocast("cuda", dtype=dtype):
                got = m(x)
            h = int8_linear(x.to(dtype), m[0].codes, m[0].scale, m[0].bias)
            assert torch.equal(got, int8_linear(h, m[1].codes, m[1].scale, m[1].bias))


def test_stream_in_inference_mode_and_out(dev):
    model = build_vggt_aggregator(depth=2, dim=128, num_heads=2, device=dev)
    frames = synthetic_frames(3, size=112, device=dev)
    one, two = FrameStream(model, 3), FrameStream(model, 3)
    with torch.inference_mode():
        a = two.step(frames[:, 0])
    assert torch.equal(a, one.step(frames[:, 0]))
    snap = two.snapshot()
    two.step(frames[:, 2])
    two.restore(snap)
    assert torch.equal(two.step(frames[:, 1]), one.step(frames[:, 1]))
    with torch.inference_mode():
        assert torch.equal(two.step(frames[:, 2]), one.step(frames[:, 2]))
    two.reset()
    assert torch.equal(two.step(frames[:, 0]), a)
