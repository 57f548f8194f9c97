"""What enable_gradients puts together, as far as it needs no GPU: token orders, refusals, modules it leaves alone. CPU only."""

import pytest
import torch
import torch.nn as nn

import ress_amd as ress
from ress_amd import training
from ress_amd.aggregator import Block, LayerScale, RoPE2D, build_vggt_aggregator
from ress_amd.kernels import LayerGrid


@pytest.mark.parametrize("frames,P,S", [(1, 20, 5), (3, 130, 5), (2, 64, 0), (5, 7, 2)])
@pytest.mark.parametrize("ordered", [False, True])
def test_orders(frames, P, S, ordered):
    """Keys: a permutation, patch tokens first; queries: special ones from a whole block on; back undoes both."""
    order = torch.randperm(P - S, generator=torch.Generator().manual_seed(0)) if ordered else None
    grid = LayerGrid(B=1, H=1, frames=frames, P=P, S=S)
    keys, k_back, queries, q_back, (lo, hi) = training._orders(grid, order, torch.device("cpu"))
    n = frames * P
    assert sorted(keys.tolist()) == list(range(n))
    within = order if ordered else torch.arange(P - S)
    assert keys[: frames * (P - S)].tolist() == [f * P + S + int(j) for f in range(frames) for j in within]
    assert keys[frames * (P - S):].tolist() == [f * P + j for f in range(frames) for j in range(S)]
    assert torch.equal(keys[k_back], torch.arange(n)) and torch.equal(queries[q_back], torch.arange(n))
    assert lo == frames * (P - S) and (hi % 128 == 0 if S else hi == lo) and hi - lo < 128
    assert len(queries) == hi + frames * S and not set(q_back.tolist()) & set(range(lo, hi))


def test_gather_and_scatter_gradients():
    grid = LayerGrid(B=1, H=2, frames=2, P=9, S=2)
    keys, k_back, queries, q_back, pad = training._orders(grid, None, torch.device("cpu"))
    x = torch.randn(1, 2, 18, 3, dtype=torch.float64, requires_grad=True)

    def through(t):  # gathered, something done to each place that keeps copies apart from the rest, scattered
        y = training._Gather.apply(t, queries, q_back, pad)
        return training._Scatter.apply(y * y, queries, q_back, pad)

    assert torch.autograd.gradcheck(through, x)
    assert torch.autograd.gradcheck(lambda t: training._Gather.apply(t, keys, k_back, (0, 0)), x)
    assert torch.equal(through(x), x * x)


def test_a_model_without_blocks_is_refused():
    with pytest.raises(TypeError, match="neither blocks"):
        ress.enable_gradients(nn.Linear(4, 4))


def test_heads_that_the_kernels_do_not_take_are_refused():
    model = build_vggt_aggregator(depth=1, dim=64, num_heads=2, device="cpu", wire=False)
    with pytest.raises(ValueError, match="heads of 64 or 128"):
        ress.enable_gradients(model)
    assert not any(getattr(m, "gradients", False) for m in model.modules())


def test_switches():
    model = build_vggt_aggregator(depth=1, dim=128, num_heads=2, device="cpu")
    assert ress.enable_gradients(model) is model
    agg = model.aggregator
    assert agg.frame_blocks[0].gradients and agg.frame_blocks[0].attn.gradients and agg.global_blocks[0].attn.differentiable
    assert agg.global_blocks[0].attn.forward.config()["differentiable"] is True
    ress.apply_sparse_vggt(model, sparse_ratio=0.5)
    assert agg.global_blocks[0].attn.forward.config()["differentiable"] is True  # a mode does not take it back
    ress.enable_gradients(model, on=False)
    assert not agg.frame_blocks[0].gradients and agg.global_blocks[0].attn.forward.config()["differentiable"] is False


def test_without_gradients_a_block_runs_as_before(monkeypatch):
    block = Block(128, 2, 2.0, RoPE2D())
    x = torch.randn(1, 6, 128)
    pos = torch.randint(0, 4, (1, 6, 2))
    monkeypatch.setattr(training, "block_forward", lambda *a: pytest.fail("without gradients"))
    monkeypatch.setattr(training, "attention_forward", lambda *a: pytest.fail("without gradients"))
    with torch.no_grad():
        want = block(x, pos)
        block.gradients = block.attn.gradients = True
        assert torch.equal(block(x, pos), want)


def test_bare_modules():
    norm = nn.LayerNorm(8)
    assert training._bare(norm, nn.LayerNorm) and not training._bare(nn.Identity(), nn.LayerNorm)
    handle = norm.register_forward_hook(lambda *a: None)
    assert not training._bare(norm, nn.LayerNorm)
    handle.remove()
    assert training._bare(norm, nn.LayerNorm)

    class Other(LayerScale):
        pass

    assert not training._bare(Other(8), LayerScale)
