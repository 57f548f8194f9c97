"""ress_amd.block_attention and its gradients against the definition in 64 bits (tests/attention_reference.py)."""

import math

import pytest
import torch

import ress_amd as ress
from attention_reference import check, reference, visible

pytestmark = pytest.mark.gpu
NAMES = ("out", "dq", "dk", "dv")


def make(B, Hq, Hk, Tq, Tk, D, dt, seed=0, layout="heads", size=1.0):
    g = torch.Generator().manual_seed(seed)

    def one(H, T, off):
        x = (torch.randn(B, H, T, D, generator=g) * size + off).to(dt)
        if layout == "tokens":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "packed":  # among others, as in a projection's output
            y = torch.zeros(B, T, 3, H, D, dtype=dt)
            y[:, :, 1] = x.transpose(1, 2)
            return y.cuda()[:, :, 1].transpose(1, 2).requires_grad_()
        return x.cuda().requires_grad_()

    q, k, v = one(Hq, Tq, 0.0), one(Hk, Tk, 0.3), one(Hk, Tk, 0.5)
    do = (torch.randn(B, Hq, Tq, D, generator=g) * 0.1).to(dt).cuda()
    return q, k, v, do


def run(q, k, v, do, **kw):
    out = ress.block_attention(q, k, v, **kw)
    return (out, *torch.autograd.grad(out, (q, k, v), do))


def compare(q, k, v, do, causal=False, q_lens=None, k_lens=None, block_map=None, scale=None):
    dev = q.device
    lens = {n: None if x is None else torch.tensor(x, dtype=torch.int32, device=dev) for n, x in (("q_lens", q_lens), ("k_lens", k_lens))}
    got = run(q, k, v, do, causal=causal, block_map=block_map, scale=scale, **lens)
    see = visible(q.shape[0], q.shape[1], q.shape[2], k.shape[2], causal, q_lens, k_lens, block_map)
    check(got, reference(q, k, v, see, scale, do), NAMES)
    with torch.no_grad():  # without gradients: the same bits
        alone = ress.block_attention(q, k, v, causal=causal, block_map=block_map, scale=scale, **lens)
    assert torch.equal(alone, got[0])
    return got


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (1, 64), (2, 65), (31, 33), (64, 1), (127, 129), (128, 64), (129, 200), (300, 511)])
def test_sizes(dev, dt, D, Tq, Tk):
    compare(*make(2, 2, 2, Tq, Tk, D, dt))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(4, 1), (6, 3), (8, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_shared_heads(dev, dt, D, Hq, Hk, causal):
    compare(*make(2, Hq, Hk, 150, 170, D, dt, layout="tokens"), causal=causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (5, 5), (64, 64), (130, 130), (200, 333), (333, 200), (1, 300), (300, 1)])
def test_causal(dev, D, Tq, Tk):
    """Rows before the first key (Tq > Tk) see nothing."""
    compare(*make(1, 2, 1, Tq, Tk, D, torch.bfloat16), causal=True)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(dev, dt, D, causal):
    q_lens, k_lens = [0, 1, 200, 129, 77, 200], [5, 0, 260, 64, 193, 1]
    q, k, v, do = make(6, 4, 2, 200, 260, D, dt, layout="packed")
    with torch.no_grad():  # what lies past the lengths reaches nothing
        for b, (m, n) in enumerate(zip(q_lens, k_lens)):
            q[b, :, m:] = math.nan
            do[b, :, m:] = math.inf
            k[b, :, n:] = math.inf
            v[b, :, n:] = math.nan
    got = compare(q, k, v, do, causal=causal, q_lens=q_lens, k_lens=k_lens)
    for b, (m, n) in enumerate(zip(q_lens, k_lens)):
        for x, at in zip(got, (m, m, n, n)):
            assert (x[b, :, at:] == 0).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", ["plain", "causal", "lengths", "shared"])
def test_maps(dev, dt, D, case):
    B, Hq, Hk, Tq, Tk = 2, 4, 2, 517, 700
    q, k, v, do = make(B, Hq, Hk, Tq, Tk, D, dt)
    g = torch.Generator().manual_seed(3)
    m = torch.rand(1 if case == "shared" else B, 1 if case == "shared" else Hq, 5, 11, generator=g) < 0.4
    m[0, 0, 2] = False   # rows that see nothing
    m[:, 0, :, 4] = False
    m[0, -1, 0] = True
    kw = {"causal": dict(causal=True), "lengths": dict(q_lens=[517, 300], k_lens=[650, 129])}.get(case, {})
    compare(q, k, v, do, block_map=m.to(dev), **kw)


def test_a_map_of_bytes_and_strides(dev):
    q, k, v, do = make(1, 2, 2, 256, 256, 64, torch.bfloat16)
    m = (torch.rand(1, 2, 4, 2, generator=torch.Generator().manual_seed(1)) < 0.6).to(dev)
    want = run(q, k, v, do, block_map=m.transpose(2, 3).contiguous())
    got = run(q, k, v, do, block_map=m.to(torch.uint8).mul(7).transpose(2, 3))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_a_map_drops_reaches_nothing(dev):
    q, k, v, do = make(1, 2, 2, 256, 320, 64, torch.bfloat16)
    m = torch.tensor([[1, 0, 1, 0, 1], [1, 0, 0, 0, 1]], dtype=torch.bool, device=dev)[None, None]
    want = run(q, k, v, do, block_map=m)
    with torch.no_grad():
        k[:, :, 64:128], v[:, :, 64:128], k[:, :, 192:256], v[:, :, 192:256] = math.nan, math.inf, math.inf, math.nan
    got = run(q, k, v, do, block_map=m)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert (got[2][:, :, 64:128] == 0).all() and (got[3][:, :, 192:256] == 0).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk,Tq,Tk", [(1, 1, 3, 17000), (2, 2, 130, 3000), (3, 1, 1, 20000), (2, 1, 9000, 70), (8, 1, 2000, 1), (1, 1, 17000, 65)])
@pytest.mark.parametrize("kind", ["dense", "causal", "map", "lengths"])
def test_few_rows_or_few_keys(dev, dt, D, Hq, Hk, Tq, Tk, kind):
    """Long axes that are cut into parts, some of which see nothing."""
    q, k, v, do = make(1, Hq, Hk, Tq, Tk, D, dt)
    kw = {}
    if kind == "causal":
        kw["causal"] = True
    if kind == "lengths":
        kw.update(q_lens=[max(1, Tq - Tq // 3)], k_lens=[max(1, Tk // 5)])
    if kind == "map":
        g = torch.Generator().manual_seed(2)
        kw["block_map"] = (torch.rand(1, Hq, -(-Tq // 128), -(-Tk // 64), generator=g) < 0.05).to(dev)
    compare(q, k, v, do, **kw)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_large_scores(dev, dt):
    """Rows that one key takes whole, scores far from zero on both sides, running maxima that move many times."""
    q, k, v, do = make(1, 2, 2, 200, 700, 64, dt, size=3.0)
    with torch.no_grad():
        k *= torch.linspace(0.1, 4.0, 700, device=dev)[:, None]
        q[:, :, 50:] -= 4.0
    compare(q, k, v, do)
    compare(q, k, v, do, scale=0.01)


def test_small_gradients_in_fp16(dev):
    """Gradients of the scores far below fp16's smallest number still reach dq and dk."""
    q, k, v, do = make(1, 2, 2, 256, 2000, 64, torch.float16)
    do = (do * 1e-2).to(torch.float16)
    got = compare(q, k, v, do)
    see = visible(1, 2, 256, 2000)
    for name, x in zip(NAMES, got):
        want = reference(q, k, v, see, None, do)[name][0]
        floor = 2.0 ** -25  # the result's own smallest step
        rel = ((x.double() - want).norm() / want.norm()).item()
        assert rel <= 2.0 ** -10 + floor * math.sqrt(want.numel()) / want.norm().item(), (name, rel)


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(dev, causal):
    """The directional derivative of sum(out * do) in 64 bits, by the definition's differences."""
    q, k, v, do = make(1, 2, 1, 70, 90, 64, torch.bfloat16)
    got = run(q, k, v, do, causal=causal)
    see = visible(1, 2, 70, 90, causal).to(dev)
    g = torch.Generator().manual_seed(9)

    def value(qkv):
        q_, k_, v_ = qkv
        s = (q_ @ k_.repeat_interleave(2, 1).transpose(2, 3).contiguous()) / 8.0
        return (torch.softmax(s.masked_fill(~see, -math.inf), -1) @ v_.repeat_interleave(2, 1) * do.double()).sum()

    at = [t.detach().double() for t in (q, k, v)]
    for n in range(3):
        d = torch.randn(at[n].shape, generator=g).to(dev).double()
        h = 1e-4
        diff = (value([t + h * d if i == n else t for i, t in enumerate(at)])
                - value([t - h * d if i == n else t for i, t in enumerate(at)])) / (2 * h)
        # the bounds of each element, as independent errors would be far below their sum
        bound = (reference(q, k, v, see.cpu(), None, do)[NAMES[n + 1]][1] * d.abs()).sum()
        assert (got[n + 1].double() * d).sum().sub(diff).abs() <= bound + 1e-6 * diff.abs()


def test_strides(dev):
    """Operands that are views, expanded, unaligned or of a single token: the contiguous call's bits."""
    q, k, v, do = (t.detach() for t in make(2, 2, 2, 100, 100, 64, torch.bfloat16))
    want = run(*(t.clone().requires_grad_() for t in (q, k, v)), do)
    wide = torch.randn(2, 2, 100, 80, device=dev).bfloat16()

    def inside(t, at):
        w = wide.clone()
        w[..., at:at + 64] = t
        return w[..., at:at + 64]

    for at in (8, 3):
        got = run(*(inside(t, at).requires_grad_() for t in (q, k, v)), inside(do, at))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    every = do[:, :, :1].expand(-1, -1, 100, -1)
    a = run(*(t.clone().requires_grad_() for t in (q, k, v)), every)
    b = run(*(t.clone().requires_grad_() for t in (q, k, v)), every.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    ke = k[:1, :1].clone().requires_grad_()
    out = ress.block_attention(q, ke.expand(2, 2, -1, -1), v)
    got = torch.autograd.grad(out, ke, do)[0]
    kc = ke.detach().expand(2, 2, -1, -1).contiguous().requires_grad_()
    full = torch.autograd.grad(ress.block_attention(q, kc, v), kc, do)[0]
    assert torch.equal(got, full.sum((0, 1), keepdim=True))


def test_empty(dev):
    for B, Tq, Tk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        q = torch.randn(B, 2, Tq, 64, device=dev).bfloat16().requires_grad_()
        k = torch.randn(B, 2, Tk, 64, device=dev).bfloat16().requires_grad_()
        v = k.detach().clone().requires_grad_()
        got = run(q, k, v, torch.ones_like(q))
        for x, like in zip(got, (q, q, k, v)):
            assert x.shape == like.shape and (x == 0).all()


def test_not_finite_values_reach_the_rows_that_see_them(dev):
    q, k, v, do = make(1, 1, 1, 256, 256, 64, torch.bfloat16)
    m = torch.tensor([[1, 1, 0, 0], [0, 0, 1, 1]], dtype=torch.bool, device=dev)[None, None]
    with torch.no_grad():
        v[0, 0, 70] = math.nan
    out = ress.block_attention(q, k, v, block_map=m)
    assert out[0, 0, :128].isnan().all() and out[0, 0, 128:].isfinite().all()


def test_repeats_bit_for_bit(dev):
    q, k, v, do = make(2, 4, 2, 700, 900, 64, torch.float16)
    first = run(q, k, v, do, causal=True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, do, causal=True), first))


def test_another_stream(dev):
    q, k, v, do = make(1, 2, 2, 300, 300, 64, torch.bfloat16)
    want = run(q, k, v, do)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(q, k, v, do)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_captured(dev, dt):
    """A forward and backward pass in a graph, replayed on new inputs with eager work between."""
    q, k, v, do = make(2, 4, 2, 200, 260, 64, dt)
    lens = torch.tensor([200, 130], dtype=torch.int32, device=dev), torch.tensor([260, 64], dtype=torch.int32, device=dev)
    kw = dict(causal=True, q_lens=lens[0], k_lens=lens[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(q, k, v, do, **kw)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(q, k, v, do, **kw)
    for i in range(4):
        new = make(2, 4, 2, 200, 260, 64, dt, seed=i)
        with torch.no_grad():
            for a, b in zip((q, k, v, do), new):
                a.copy_(b)
            lens[1][1] = 64 + 40 * i
        graph.replay()
        torch.cuda.synchronize()
        want = run(*new, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_a_leafs_gradient_accumulates(dev):
    q, k, v, do = make(1, 2, 2, 100, 100, 64, torch.bfloat16)
    want = run(q, k, v, do)
    ress.block_attention(q, k, v).backward(do)
    assert torch.equal(q.grad, want[1]) and torch.equal(k.grad, want[2]) and torch.equal(v.grad, want[3])
    out = ress.block_attention(q, k.detach(), v.detach())
    assert torch.equal(torch.autograd.grad(out, q, do)[0], want[1])


def test_a_capture_beside_an_eager_result_of_the_same_leaves_is_refused(dev):
    """Refused before anything is recorded; once the eager result is gone the same capture works."""
    q, k, v, do = make(1, 2, 2, 64, 64, 64, torch.bfloat16)
    want = run(q, k, v, do)
    out = ress.block_attention(q, k, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="still alive"):
                ress.block_attention(q, k, v)
            torch.zeros(1, device=dev)
        finally:
            graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
    want = [t.detach() for t in want]
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(q, k, v, do)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("D", [64, 128])
def test_tokens_far_apart(dev, D):
    """Offsets past 2^32 bytes: operands and gradients in a buffer whose tokens lie 4 MB apart give the contiguous call's bits."""
    T, apart = 1300, 1 << 21
    wide = torch.empty(T, apart, dtype=torch.bfloat16, device=dev)
    q, k, v, do = (t.detach() for t in make(1, 2, 2, T, T, D, torch.bfloat16))
    want = run(*(t.clone().requires_grad_() for t in (q, k, v)), do, causal=True)
    far = []
    for i, t in enumerate((q, k, v, do)):
        to = wide[:, apart - (i + 1) * 2 * D:][:, :2 * D].view(T, 2, D).transpose(0, 1)[None]
        to.copy_(t)
        far.append(to)
    got = run(*(t.requires_grad_() for t in far[:3]), far[3], causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dt,u", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk", [(1, 5), (4, 14), (40, 70)])
def test_few_probabilities_are_not_rounded(dev, dt, u, D, Tq, Tk):
    """P and dS in two terms: each element is off by its own rounding and by 2^-14 of what its sums add up (two terms of 8 bits and a sign
    leave 2^-17 of a factor, exponentials, sums and delta 2^-18 each and less; P alone rounded to bf16 would leave 2^-8)."""
    q, k, v, do = make(1, 2, 2, Tq, Tk, D, dt)
    out, dq, dk, dv = run(q, k, v, do)
    q, k, v, g = (t.detach().double() for t in (q, k, v, do))
    scale = 1.0 / math.sqrt(D)
    p = (torch.matmul(q, k.transpose(2, 3)) * scale).softmax(-1)
    o = torch.matmul(p, v)
    dp = torch.matmul(g, v.transpose(2, 3))
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    size = p * (torch.matmul(g.abs(), v.abs().transpose(2, 3)) + (g.abs() * torch.matmul(p, v.abs())).sum(-1, keepdim=True))
    # a score is a sum, too: 2^-18 of its terms moves p by as much of itself, times the terms' sum
    size = size * (1 + scale * torch.matmul(q.abs(), k.abs().transpose(2, 3)))
    wide = p * (1 + scale * torch.matmul(q.abs(), k.abs().transpose(2, 3)))
    far = k.abs().amax(2, keepdim=True)
    for got, want, mag in ((out, o, torch.matmul(wide, v.abs())),
                           (dq, scale * torch.matmul(ds, k), scale * (size.sum(-1, keepdim=True) * far)),
                           (dk, scale * torch.matmul(ds.transpose(2, 3), q), scale * torch.matmul(size.transpose(2, 3), q.abs())),
                           (dv, torch.matmul(p.transpose(2, 3), g), torch.matmul(wide.transpose(2, 3), g.abs()))):
        bound = u * want.abs() + 2.0 ** -14 * mag + (2.0 ** -25 if dt is torch.float16 else 0.0)
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk,causal", [(1, 64, False), (2, 65, True), (31, 33, False), (64, 64, True), (127, 129, True), (129, 200, False)])
def test_small_sizes_of_many_heads(dev, dt, D, Tq, Tk, causal):
    """More than 2^18 probabilities: rounded ones."""
    H = 2 * ((1 << 17) // (Tq * Tk) + 1)
    compare(*make(1, H, H // 2, Tq, Tk, D, dt), causal=causal)
