"""Which modules enable_gradients does the arithmetic of in their place: those that are just what they are called, with nothing on them."""

import types

import pytest
import torch
import torch.nn as nn

import ress_amd as ress
from ress_amd import training
from ress_amd.aggregator import Block, LayerScale, RoPE2D


def on_gpu(*shape, dtype=torch.bfloat16):
    """What _norm_takes looks at of a device tensor."""
    x = torch.empty(shape, dtype=dtype, device="meta")
    return types.SimpleNamespace(is_cuda=True, dtype=dtype, shape=x.shape, numel=x.numel, dim=x.dim)


def test_a_replaced_forward():
    for module in (nn.LayerNorm(8), LayerScale(8)):
        assert training._bare(module, type(module))
        forward = module.forward
        module.forward = lambda x: forward(x) * 2.0
        assert not training._bare(module, type(module))
        del module.forward
        assert training._bare(module, type(module))


@pytest.mark.parametrize("register", [
    lambda f: nn.modules.module.register_module_forward_hook(f), lambda f: nn.modules.module.register_module_forward_pre_hook(f),
    lambda f: nn.modules.module.register_module_full_backward_hook(f), lambda f: nn.modules.module.register_module_full_backward_pre_hook(f)])
def test_global_hooks(register):
    norm = nn.LayerNorm(8)
    handle = register(lambda *a: None)
    try:
        assert not training._bare(norm, nn.LayerNorm)
    finally:
        handle.remove()
    assert training._bare(norm, nn.LayerNorm)


def test_norms_that_the_kernels_do_not_take():
    norm = nn.LayerNorm(64).bfloat16()
    assert training._norm_takes(norm, on_gpu(3, 64)) and training._norm_takes(nn.LayerNorm(64), on_gpu(3, 64))
    assert training._norm_takes(nn.LayerNorm(8192).bfloat16(), on_gpu(3, 8192))
    assert not training._norm_takes(nn.LayerNorm(8200).bfloat16(), on_gpu(3, 8200))
    assert not training._norm_takes(norm, on_gpu(3, 32))  # torch's error
    assert not training._norm_takes(norm, on_gpu(1 << 31, 64))
    assert not training._norm_takes(norm, on_gpu(3, 64, dtype=torch.float64))
    mixed = nn.LayerNorm(64).bfloat16()
    mixed.bias = nn.Parameter(torch.zeros(64))
    assert not training._norm_takes(mixed, on_gpu(3, 64))


@pytest.mark.gpu
def test_a_wide_norm_runs_as_it_is(dev):
    norm = nn.LayerNorm(8200).to(dev, torch.bfloat16)
    x = torch.randn(3, 8200, device=dev).bfloat16().requires_grad_()
    assert torch.equal(training._norm(norm, x), norm(x))


@pytest.mark.gpu
def test_a_replaced_forward_is_run(dev):
    block = Block(128, 2, 2.0, RoPE2D()).to(dev, torch.bfloat16)
    ress.enable_gradients(block)
    x, pos = torch.randn(1, 6, 128, device=dev).bfloat16(), torch.zeros(1, 6, 2, dtype=torch.int64, device=dev)
    seen = []
    for name, module in (("norm1", block.norm1), ("norm2", block.norm2), ("ls1", block.ls1), ("q_norm", block.attn.q_norm)):
        forward = module.forward
        module.forward = lambda y, forward=forward, name=name: (seen.append(name), forward(y))[1]
    block(x, pos)
    assert seen == ["norm1", "q_norm", "ls1", "norm2"]
    counted = []
    handle = nn.modules.module.register_module_forward_hook(lambda m, a, out: counted.append(type(m).__name__))
    try:
        other = Block(128, 2, 2.0, RoPE2D()).to(dev, torch.bfloat16)
        ress.enable_gradients(other)
        other(x, pos)
    finally:
        handle.remove()
    assert counted.count("LayerNorm") == 4 and counted.count("LayerScale") == 2
