"""A model's gradients through the operators with a backward pass: against the same model in 64 bits, and through the sparse layers
against the definition over the same map."""

import copy
import math

import pytest
import torch
import torch.nn.functional as F

import ress_amd as ress
from attention_reference import check, reference
from ress_amd import training
from ress_amd.aggregator import build_vggt_aggregator, synthetic_frames
from ress_amd.kernels import LayerGrid

pytestmark = pytest.mark.gpu
# A bfloat16 model of four blocks: some 24 tensors a block are rounded on the way there and back, each by 2^-8 / sqrt(3) rms at most,
# independently: sqrt(96) 2^-8 / sqrt(3) = 2.2% of a gradient's norm; twice that for what norms and softmax make of it.
MODEL_TOLERANCE = 2 * math.sqrt(96) * 2.0 ** -8 / math.sqrt(3)


def small(wire, seed=0, depth=2, scale=0.3):
    model = build_vggt_aggregator(depth=depth, dim=128, num_heads=2, seed=seed, wire=wire)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for m in model.modules():  # branches that count, and norms that are not the identity
            if hasattr(m, "gamma"):
                m.gamma.copy_(scale * (1 + 0.3 * torch.randn(m.gamma.shape, generator=g)))
            if isinstance(m, torch.nn.LayerNorm):
                m.weight.copy_(1 + 0.2 * torch.randn(m.weight.shape, generator=g))
                m.bias.copy_(0.1 * torch.randn(m.bias.shape, generator=g))
    return model


def gradients(model, images, target):
    model.zero_grad(set_to_none=True)
    out = model(images)
    (out.to(target.dtype) * target).sum().backward()
    return {n: p.grad for n, p in model.named_parameters()}, out


def test_a_dense_models_gradients(dev):
    """Every parameter's, against the plain modules in 64 bits."""
    model = small(False)
    images = synthetic_frames(3, size=70).to(torch.bfloat16)
    exact = copy.deepcopy(model).double()
    for m in exact.modules():
        if hasattr(m, "fused"):
            m.fused = False
    target = torch.randn(1, 90, 128, generator=torch.Generator().manual_seed(1)).to(dev)
    want, out64 = gradients(exact, images.double(), target.double())
    ress.enable_gradients(model)
    got, out = gradients(model, images, target)
    assert ((out.double() - out64).norm() / out64.norm()) <= MODEL_TOLERANCE
    for name, w in want.items():
        if w.norm() == 0:  # the key's bias turned by nothing: softmax does not see it
            continue
        if name.endswith("qkv.bias"):  # nor the key part of the projection's
            w, g = torch.cat([w[:128], w[256:]]), torch.cat([got[name][:128], got[name][256:]])
        else:
            g = got[name]
        assert ((g.double() - w).norm() / w.norm()) <= MODEL_TOLERANCE, name


@pytest.mark.parametrize("S", [0, 5])
@pytest.mark.parametrize("ordered", [False, True])
def test_sparse_attention(dev, S, ordered):
    """The attention over a layer's map, in storage order, with gradients of all three operands."""
    B, H, frames, hw = 2, 3, 3, 110
    P = hw + S
    grid = LayerGrid(B=B, H=H, frames=frames, P=P, S=S)
    g = torch.Generator().manual_seed(S)
    q, k, v, do = (torch.randn(B, H, frames * P, 64, generator=g).to(dev, torch.bfloat16) for _ in range(4))
    do *= 0.1
    order = torch.randperm(hw, generator=g).to(dev, torch.int32) if ordered else None
    final_map = (torch.rand(B, H, -(-frames * hw // 128), -(-frames * P // 64), generator=g) < 0.5).to(dev)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = training.sparse_attention(*leaves, final_map, grid, order)
    got = (out, *torch.autograd.grad(out, leaves, do))
    within = torch.arange(hw) if order is None else order.cpu().long()
    keys = torch.tensor([f * P + S + int(j) for f in range(frames) for j in within]
                        + [f * P + j for f in range(frames) for j in range(S)])
    see = torch.zeros(B, H, frames * P, frames * P, dtype=torch.bool)
    rows, m = keys[: frames * hw], final_map.cpu()
    part = m.repeat_interleave(128, 2)[:, :, : len(rows)].repeat_interleave(64, 3)[..., : len(keys)]
    see[:, :, rows[:, None], keys[None]] = part
    see[:, :, keys[len(rows):]] = True
    check(got, reference(q, k, v, see, None, do), ("out", "dq", "dk", "dv"))


@pytest.mark.parametrize("mode", ["sparse_vggt", "ress", "dense"])
def test_a_sparse_models_step(dev, mode):
    """A training step through wired layers: every parameter gets a gradient, the output is near the inference path's, and that is what it
    was."""
    g = torch.Generator().manual_seed(2)
    tables = tuple(torch.rand(3, 2, 2, generator=g) + 0.1 for _ in range(2))
    model = small(True)
    model._ress_calibration_tables = tables
    images = synthetic_frames(4, size=14 * 12).to(torch.bfloat16)
    if mode == "sparse_vggt":
        ress.apply_sparse_vggt(model, sparse_ratio=0.5)
    elif mode == "ress":
        ress.apply_ress(model, sparse_ratio=0.5, backbone="vggt")
    else:
        ress.apply_dense(model)
    with torch.no_grad():
        before = model(images)
        ress.enable_gradients(model)
        assert torch.equal(model(images), before)
    target = torch.randn(before.shape, generator=g).to(dev)
    got, out = gradients(model, images, target)
    assert ((out - before).float().norm() / before.float().norm()) <= MODEL_TOLERANCE
    for name, t in got.items():
        assert t is not None and torch.isfinite(t).all() and t.abs().max() > 0, name
    again, _ = gradients(model, images, target)
    blocks = [n for n in got if "blocks" in n and "bias" not in n and "weight" in n]
    assert blocks
    ress.check_layers(model)
    loss = []
    optimiser = torch.optim.SGD(model.parameters(), lr=1e-4)
    for _ in range(2):
        optimiser.zero_grad()
        out = model(images)
        (out.float() * target).mean().backward()
        optimiser.step()
        loss.append(out)
    assert all(torch.isfinite(x).all() for x in loss)


def test_recorded_output_gradients(dev):
    """retain_output_grad and the recorded outputs, which head scores are made of."""
    model = small(True, depth=1)
    from ress_amd.wiring import wire_ress_attention
    stores = [{}]
    wire_ress_attention(model, model.aggregator.global_blocks, stores)
    ress.apply_sparse_vggt(model, sparse_ratio=0.5)
    ress.enable_gradients(model)
    attn = model.aggregator.global_blocks[0].attn
    attn.retain_output_grad = True
    images = synthetic_frames(2, size=14 * 12).to(torch.bfloat16)
    model(images).float().square().mean().backward()
    o = stores[0]["value"].output
    assert o.grad is not None and torch.isfinite(o.grad).all() and o.grad.abs().max() > 0
    assert 0.0 <= stores[0]["value"].sparsity < 1.0


def test_modules_with_hooks_are_run(dev):
    """A hook on a norm, or another module in its place, sees every call."""
    model = small(False, depth=1)
    ress.enable_gradients(model)
    seen = []
    for block in model.aggregator.frame_blocks:
        block.norm2.register_forward_hook(lambda m, a, out: seen.append("norm2"))
        block.ls1.register_forward_hook(lambda m, a, out: seen.append("ls1"))
        block.attn.q_norm.register_forward_hook(lambda m, a, out: seen.append("q_norm"))
    model(synthetic_frames(1, size=70).to(torch.bfloat16)).float().sum().backward()
    assert seen == ["q_norm", "ls1", "norm2"]


def test_a_32_bit_model_under_autocast(dev):
    model = small(False, depth=1).float()
    ress.enable_gradients(model)
    images = synthetic_frames(2, size=70)
    with torch.autocast("cuda", torch.bfloat16):
        out = model(images)
    out.float().square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        model(images)


def test_the_operators_in_a_row(dev):
    """Norm, projection, head norms, rotation, attention, residual norm as a block runs them, against the same in 64 bits: one block's 24
    roundings."""
    model = small(False, depth=1)
    ress.enable_gradients(model)
    block = model.aggregator.frame_blocks[0]
    exact = copy.deepcopy(block).double()
    exact.gradients = exact.attn.gradients = exact.attn.fused = False
    x = torch.randn(2, 150, 128, generator=torch.Generator().manual_seed(0)).to(dev, torch.bfloat16).requires_grad_()
    pos = torch.randint(0, 37, (2, 150, 2), generator=torch.Generator().manual_seed(1)).to(dev)
    dy = torch.randn(2, 150, 128, generator=torch.Generator().manual_seed(2)).to(dev)
    y = block(x, pos)
    got, = torch.autograd.grad(y, x, dy.to(y.dtype))
    x64 = x.detach().double().requires_grad_()
    want, = torch.autograd.grad(exact(x64, pos), x64, dy.to(y.dtype).double())
    assert ((got.double() - want).norm() / want.norm()) <= MODEL_TOLERANCE / 2
    assert F.cosine_similarity(got.double().flatten(), want.flatten(), dim=0) > 0.999


def test_a_captured_row_of_operators(dev):
    """Residual norm, rotation and causal attention, there and back, in one graph beside eager work of the same kind: every replay as the
    eager pass on the same inputs."""
    g = torch.Generator().manual_seed(4)
    rope = ress.RotaryTable(64, 300, base=10000.0, axes=1, device=dev, layout="interleaved")
    pos = torch.arange(130, device=dev)

    def inputs(seed):
        g.manual_seed(seed)
        shapes = ((2, 130, 128), (2, 130, 128), (128,), (128,), (128,))
        return [torch.randn(s, generator=g).to(dev, torch.bfloat16).requires_grad_() for s in shapes]

    def run(x, branch, gamma, weight, bias):
        h, n = ress.add_layer_norm(x, branch, gamma, weight, bias)
        q, k = (t.view(2, 130, 2, 64).transpose(1, 2) for t in (n, h))
        q, k = ress.rotate((q, k), pos, rope)
        out = ress.block_attention(q, k, h.view(2, 130, 2, 64).transpose(1, 2), causal=True)
        return (out, *torch.autograd.grad(out, (x, branch, gamma, weight, bias), torch.ones_like(out)))

    mine = inputs(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(*mine)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*mine)
    for seed in range(4):
        new = inputs(seed + 1)
        with torch.no_grad():
            for a, b in zip(mine, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run(*new))), seed


def test_positions_outside_a_models_table_are_reported(dev):
    model = small(False, depth=1)
    ress.enable_gradients(model)
    block = model.aggregator.frame_blocks[0]
    x = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=dev)
    block(x, torch.full((1, 4, 2), 7, device=dev))
    ress.check_layers(model)
    block(x, torch.full((1, 4, 2), 1 << 20, device=dev))
    with pytest.raises(RuntimeError, match="outside the rotation table"):
        ress.check_layers(model)
    ress.check_layers(model)


def test_a_model_that_has_not_run_is_not_captured(dev):
    model = small(False, depth=1)
    ress.enable_gradients(model)
    block = model.aggregator.frame_blocks[0]
    x, pos = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=dev), torch.zeros(1, 4, 2, dtype=torch.int64, device=dev)
    qkv = torch.zeros(1, 4, 384, dtype=torch.bfloat16, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="once before a graph capture"):
                training.normed_and_turned(block.attn, qkv, pos, 2)
            x.add_(1.0)
        finally:
            graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.isfinite(block(x, pos)).all()
