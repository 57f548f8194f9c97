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


@pytest.mark.parametrize("n", [1, 40, 56])
@pytest.mark.parametrize("length", [-(1 << 31), -1000, -1, 1000, (1 << 31) - 1])
def test_lengths_changed_from_outside(dev, n, length):
    """A length that no append left is taken as none or as what the slot's pages hold; other slots stay as they are."""
    c = PagedKVCache(12, 2, max_seqs=3, max_len=256, device=dev)
    x, new, q = _rand((3, 2, 200, 64), dev, 0), _rand((3, 2, n, 64), dev, 1), _rand((3, 2, n, 64), dev, 2)
    c.append(x, x)
    for s in range(3):
        c.reserve(s, 256)
    tails = c.tail_k[[0, 2]].clone(), c.tail_v[[0, 2]].clone(), c.tail_top[[0, 2]].clone()
    pages = c.table[[0, 2], :3].long()
    codes = c.k_codes[pages].clone(), c.v_codes[pages].clone(), c.k_scale[pages].clone(), c.v_scale[pages].clone()
    want = c.attend(q, causal=True)
    c.lens[1] = length
    for causal in (False, True):
        got = c.attend(q, causal=causal)
        if length < 0:
            assert (got[1] == 0).all()
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    k, v = c.read(n)
    if length < 0:
        assert (k[1] == 0).all() and (v[1] == 0).all()
    c.append(new[1:2], new[1:2], slots=[1])
    assert int(c.lens[1]) == (min(n, 256) if length < 0 else 256)
    if length > 0:
        with pytest.raises(RuntimeError, match="dropped"):
            c.check()
    c.check()
    assert torch.equal(c.attend(q, causal=True)[[0, 2]], want[[0, 2]])
    for a, b in zip(tails, (c.tail_k[[0, 2]], c.tail_v[[0, 2]], c.tail_top[[0, 2]])):
        assert torch.equal(a, b)
    for a, b in zip(codes, (c.k_codes[pages], c.v_codes[pages], c.k_scale[pages], c.v_scale[pages])):
        assert torch.equal(a, b)
    assert c.held.tolist() == [4, 4, 4] and c.lens.tolist()[::2] == [200, 200]
