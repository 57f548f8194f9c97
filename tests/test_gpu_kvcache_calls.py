"""Calls of the paged cache that the documentation allows or refuses, on the GPU."""

import pytest
import torch

from kvcache_oracle import attention, held, tolerance
from ress_amd.kvcache import PAGE, PagedKVCache, RotaryTable

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


def _filled(dev, H, D, lens, dtype=BF16, codes="int8"):
    c = PagedKVCache(sum(-(-(L + 200) // PAGE) for L in lens), H, D, max_seqs=len(lens), dtype=dtype, codes=codes, device=dev)
    for b, L in enumerate(lens):
        if L:
            g = torch.Generator().manual_seed(b)
            k, v = (torch.randn(1, H, L, D, generator=g).to(dev, dtype) for _ in range(2))
            c.append(k, v, slots=[b])
    return c


def _check(c, q, got, causal=False, scale=None):
    for b in range(q.shape[0]):
        k, v = held(c, b)
        want, size, spread = attention(q[b], k, v, q.shape[2], causal, scale)
        err = (got[b].double().cpu() - want).abs()
        tol = tolerance(want, size, spread, q.dtype, k.shape[1])
        assert (err <= tol).all(), (b, float((err / tol).max()))


@pytest.mark.parametrize("H,G,n", [(3, 1, 7), (5, 3, 1), (1, 7, 5), (3, 5, 9), (7, 3, 40), (1, 40, 1), (2, 33, 3)])
@pytest.mark.parametrize("dtype,codes,D", [(BF16, "int8", 64), (torch.float16, "fp8", 128)])
def test_odd_heads(dev, dtype, codes, D, H, G, n):
    """Heads and groups that are no powers of two: rows of a tile belong to several tokens, tiles to several heads."""
    c = _filled(dev, H, D, [700, 65, 30], dtype, codes)
    q = torch.randn(3, H * G, n, D, generator=torch.Generator().manual_seed(9)).to(dev, dtype)
    for causal in (False, True):
        for scale in (None, 0.05):
            _check(c, q, c.attend(q, causal=causal, scale=scale), causal, scale)


@pytest.mark.parametrize("dtype,codes,D", [(BF16, "int8", 64), (torch.float16, "int8", 128)])
@pytest.mark.parametrize("n", [20, 90, 300])
@pytest.mark.parametrize("L", [500, 6000])
def test_queries_that_are_not_finite(dev, dtype, codes, D, n, L):
    """Reach their own rows and no others, whatever rows share a tile, a wave or a register with them."""
    c = _filled(dev, 2, D, [L], dtype, codes)
    q = torch.randn(1, 4, n, D, generator=torch.Generator().manual_seed(9)).to(dev, dtype)
    want = c.attend(q, causal=True)
    for bad in (float("nan"), -float("nan"), float("inf"), -float("inf")):
        for i in (0, 3, 17):
            p = q.clone()
            p[0, 1, i, 5] = bad
            got = c.attend(p, causal=True)
            rest = torch.ones(1, 4, n, dtype=torch.bool, device=dev)
            rest[0, 1, i] = False
            assert torch.equal(got[rest], want[rest])
            assert bad == bad or got[0, 1, i].isnan().all()


def test_expanded_operands(dev):
    """Views that repeat rows, heads and sequences: as their copies do."""
    x = _rand((1, 1, 1, 64), dev, 3)
    a, b = (PagedKVCache(16, 2, max_seqs=2, device=dev) for _ in range(2))
    rope = RotaryTable(64, 300, axes=1, device=dev)
    pos = torch.arange(150, device=dev)[None]
    wide = x.expand(2, 2, 150, 64)
    qa = a.append(wide, wide, pos=pos.expand(2, 150), rope=rope, q=x.expand(2, 4, 150, 64))
    qb = b.append(wide.contiguous(), wide.contiguous(), pos=pos.repeat(2, 1), rope=rope, q=x.repeat(2, 4, 150, 1))
    assert torch.equal(qa, qb)
    for t, u in zip(a.read(150), b.read(150)):
        assert torch.equal(t, u)
    for n in (4, 70):
        got = a.attend(x.expand(2, 4, n, 64), causal=True)
        assert torch.equal(got, b.attend(x.repeat(2, 4, n, 1), causal=True))
        out = torch.full((2, n, 3, 4, 64), 9.0, dtype=BF16, device=dev)
        assert torch.equal(a.attend(x.expand(2, 4, n, 64), causal=True, out=out[:, :, 1].transpose(1, 2)), got)
        assert (out[:, :, 0] == 9).all() and (out[:, :, 2] == 9).all()


def test_captured_padded_steps(dev):
    """Counts and slots that live on the device: a graph's replays append what they say then."""
    eager, c = (PagedKVCache(24, 2, max_seqs=4, device=dev) for _ in range(2))
    x = _rand((2, 2, 30, 64), dev, 1)
    counts = torch.tensor([30, 7], dtype=torch.int32, device=dev)
    batch = c.slots([3, 1])
    for s in (3, 1):
        c.reserve(s, 300)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append(x, x, slots=batch, new_lens=counts)
        out = c.attend(x, slots=batch, new_lens=counts, causal=True)
    for i, m in enumerate(([30, 7], [1, 0], [0, 30], [29, 30], [30, 30])):
        x.copy_(_rand((2, 2, 30, 64), dev, 10 + i))
        counts.copy_(torch.tensor(m, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager.append(x, x, slots=[3, 1], new_lens=m)
        want = eager.attend(x, slots=[3, 1], new_lens=m, causal=True)
        assert eager.lengths() == c.lens.tolist()
        for s in (3, 1):
            for a, b in zip(held(eager, s), held(c, s)):
                assert torch.equal(a, b)
        assert (out.double() - want.double()).abs().max() <= 2.0 ** -8 * want.double().abs().max().clamp(min=1)
        assert (out[0, :, m[0]:] == 0).all() and (out[1, :, m[1]:] == 0).all()
    c.check()


@pytest.mark.parametrize("n", [1, 40, 100])
@pytest.mark.parametrize("bad", [-1, 3, 1 << 30, -(1 << 31)])
def test_slots_outside_the_cache(dev, n, bad):
    """A batch whose numbers on the device are changed: such a row appends nothing and sees nothing, and is reported; the
    other rows are as ever. (Lists are checked on the host.)"""
    a, b = (_filled(dev, 2, 64, [100, 5000, 30]) for _ in range(2))
    x, q = _rand((2, 2, n, 64), dev, 1), _rand((2, 4, n, 64), dev, 2)
    batch = a.slots([0, 1])
    for c in (a, b):
        c.reserve(1, 5200)
    batch.tensor[0] = bad

    def reported():
        with pytest.raises(RuntimeError, match="slot lies outside"):
            a.check()
        a.check()

    a.append(x, x, slots=batch)
    reported()
    b.append(x[1:], x[1:], slots=[1])
    assert a.lens.tolist() == b.lens.tolist() == [100, 5000 + n, 30]
    got, want = a.attend(q, slots=batch, causal=True), b.attend(q, slots=[0, 1], causal=True)
    reported()
    assert (got[0] == 0).all() and torch.equal(got[1], want[1])
    k, v = a.read(n, slots=batch)
    reported()
    assert (k[0] == 0).all() and (v[0] == 0).all() and torch.equal(k[1], b.read(n, slots=[1])[0][0])
    for s in range(3):
        for t, u in zip(held(a, s), held(b, s)):
            assert torch.equal(t, u)
