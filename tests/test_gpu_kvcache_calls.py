"""Calls of the paged cache that the documentation allows or refuses, on the GPU."""

import pytest
import torch

from ress_amd.kvcache import PAGE, PagedKVCache

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _rand(shape, dev, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dev, BF16)


def test_reserve_inside_a_capture(dev):
    """Refused, and pages and later appends are as if it had not been called."""
    c = PagedKVCache(8, 1, max_seqs=2, device=dev)
    x = _rand((1, 1, 300, 64), dev, 0)
    c.append(x[:, :, :10], x[:, :, :10])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(x[:, :, :4])
        with pytest.raises(RuntimeError, match="not inside a graph capture"):
            c.reserve(0, 200)
    assert c.free_pages() == 7
    c.append(x, x)
    c.check()
    assert c.lengths() == [310, 0] and c.held.tolist() == [5, 0]
    graph.replay()
    torch.cuda.synchronize()


def test_slots_in_every_form(dev):
    c, d = (PagedKVCache(8, 1, max_seqs=2, device=dev) for _ in range(2))
    x = _rand((1, 1, 70, 64), dev, 0)
    c.append(x, x)
    c.append(x, x, slots=torch.tensor([1]))
    c.check()
    assert c.lengths() == [70, 70]
    d.append(x, x)
    d.append(x, x, slots=[1])
    assert torch.equal(c.attend(x[:, :, :3], slots=torch.tensor([1], device=dev)), d.attend(x[:, :, :3], slots=[1]))
