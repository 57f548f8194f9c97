"""What the operators with gradients refuse in Python, before anything is launched."""

import math

import pytest
import torch

import ress_amd as ress

pytestmark = pytest.mark.gpu


def t(dev, *shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype, device=dev)


def test_attention(dev):
    q, k = t(dev, 2, 4, 200, 64), t(dev, 2, 2, 300, 64)
    ok = torch.ones(2, 4, 2, 5, dtype=torch.bool, device=dev)
    ress.block_attention(q, k, k, block_map=ok)
    for args, kw, error, msg in [
        ((q.float(), k, k), {}, TypeError, "bfloat16 or float16"),
        ((q, k.half(), k), {}, ValueError, "like q"),
        ((q, k, k.cpu()), {}, RuntimeError, "device tensor"),
        ((q[0], k, k), {}, ValueError, r"\(B, heads"),
        ((t(dev, 2, 4, 200, 80), t(dev, 2, 2, 300, 80), t(dev, 2, 2, 300, 80)), {}, ValueError, "head_dim must be"),
        ((q, k, k[:, :, :200]), {}, ValueError, "k and v must be"),
        ((q, k[:1], k[:1]), {}, ValueError, "k and v must be"),
        ((t(dev, 2, 3, 200, 64), k, k), {}, ValueError, "multiple of k's heads"),
        ((q, k[:, :0], k[:, :0]), {}, ValueError, "multiple of k's heads"),
        ((q, k, k), dict(block_map=ok[:, :, :1]), ValueError, "block_map must be"),
        ((q, k, k), dict(block_map=ok.float()), ValueError, "bool or uint8"),
        ((q, k, k), dict(block_map=ok.cpu()), ValueError, "bool or uint8"),
        ((q, k, k), dict(block_map=ok[:, :3]), ValueError, "block_map must be"),
        ((q, k, k), dict(scale=0.0), ValueError, "scale"),
        ((q, k, k), dict(scale=math.nan), ValueError, "scale"),
        ((q, k, k), dict(q_lens=[1]), ValueError, "q_lens"),
        ((q, k, k), dict(q_lens=[1, 201]), ValueError, "q_lens"),
        ((q, k, k), dict(k_lens=[-1, 3]), ValueError, "k_lens"),
        ((q, k, k), dict(k_lens=torch.tensor([1, 2], device=dev)), ValueError, "int32"),
        ((q, k, k), dict(k_lens=torch.tensor([1, 2], dtype=torch.int32)), ValueError, "int32"),
    ]:
        with pytest.raises(error, match=msg):
            ress.block_attention(*args, **kw)


def test_norms(dev):
    x, w = t(dev, 3, 64), t(dev, 64)
    for call, error, msg in [
        (lambda: ress.layer_norm(x.double()), TypeError, "bfloat16, float16 or float32"),
        (lambda: ress.layer_norm(t(dev, 3, 8193)), ValueError, "last dim"),
        (lambda: ress.layer_norm(t(dev, 3, 0)), ValueError, "last dim"),
        (lambda: ress.layer_norm(x, w[:63]), ValueError, "weight must be"),
        (lambda: ress.layer_norm(x, w.half()), ValueError, "weight must be"),
        (lambda: ress.layer_norm(x, w, w.float()), ValueError, "one type"),
        (lambda: ress.layer_norm(x, w.cpu()), ValueError, "weight must be"),
        (lambda: ress.layer_norm(x, eps=-1.0), ValueError, "eps"),
        (lambda: ress.layer_norm(x, eps=math.nan), ValueError, "eps"),
        (lambda: ress.add_layer_norm(x, None), ValueError, "branch"),
        (lambda: ress.add_layer_norm(x, x[:2]), ValueError, "branch must be"),
        (lambda: ress.add_layer_norm(x, x.float()), ValueError, "branch must be"),
        (lambda: ress.add_layer_norm(x, x, w.float(), w, w), ValueError, "one type"),
    ]:
        with pytest.raises(error, match=msg):
            call()


def test_rotations(dev):
    x, pos = t(dev, 2, 3, 5, 64), torch.arange(5, device=dev)
    one, two = (ress.RotaryTable(64, 8, axes=a, device=dev) for a in (1, 2))
    for call, error, msg in [
        (lambda: ress.rotate(x.float(), pos, one), TypeError, "bfloat16 or float16"),
        (lambda: ress.rotate(t(dev, 2, 3, 5, 128), pos, one), ValueError, "x must be"),
        (lambda: ress.rotate((x, x, x), pos, one), ValueError, "one or two"),
        (lambda: ress.rotate((), pos, one), ValueError, "one or two"),
        (lambda: ress.rotate((x, x[:1]), pos, one), ValueError, "turned together"),
        (lambda: ress.rotate((x, x.half()), pos, one), ValueError, "turned together"),
        (lambda: ress.rotate(x, pos.float(), one), ValueError, "whole numbers"),
        (lambda: ress.rotate(x, pos.cpu(), one), ValueError, "whole numbers"),
        (lambda: ress.rotate(x, pos[:4], one), ValueError, "whole numbers"),
        (lambda: ress.rotate(x, pos, two), ValueError, "whole numbers"),
        (lambda: ress.rotate(x, pos, ress.RotaryTable(64, 8, axes=1, device="cpu")), ValueError, "rope is on"),
    ]:
        with pytest.raises(error, match=msg):
            call()


def test_second_derivatives_are_refused(dev):
    x = torch.randn(3, 64, device=dev, requires_grad=True)
    g, = torch.autograd.grad(ress.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_lists_inside_a_capture(dev):
    q = t(dev, 2, 2, 10, 64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="made before it"):
                ress.block_attention(q, q, q, k_lens=[3, 4])
            torch.zeros(1, device=dev)
        finally:
            graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
