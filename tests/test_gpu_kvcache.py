"""The paged 8-bit key/value cache: what append puts into it, read, and attention over it, against 64 bits."""

import math

import pytest
import torch

from kvcache_oracle import PAGE, attention, half_step, held, tolerance
from ress_amd.kvcache import PagedKVCache, RotaryTable

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
KINDS = [(BF16, "int8", 64), (BF16, "fp8", 128), (F16, "int8", 128), (F16, "fp8", 64)]


def _rand(shape, dtype, dev, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * gain).to(dtype).to(dev)


def _cache(dev, H=2, D=64, S=1, tokens=1024, dtype=BF16, codes="int8"):
    return PagedKVCache(S * (tokens // PAGE + 1), H, D, max_seqs=S, max_len=tokens, dtype=dtype, codes=codes, device=dev)


def _filled(dev, lens, H=2, D=64, dtype=BF16, codes="int8", seed=0, room=64):
    S, T = len(lens), max(lens + [1])
    c = _cache(dev, H, D, S, T + room, dtype, codes)
    k = _rand((S, H, T, D), dtype, dev, seed) + _rand((1, H, 1, D), dtype, dev, seed + 1)
    v = _rand((S, H, T, D), dtype, dev, seed + 2) + _rand((1, H, 1, D), dtype, dev, seed + 3)
    c.append(k, v, new_lens=lens)
    return c, k, v


# ---- append -----------------------------------------------------------------
@pytest.mark.parametrize("dtype,codes,D", KINDS)
@pytest.mark.parametrize("n", [1, 63, 64, 65, 200])
def test_held_values(dev, dtype, codes, D, n):
    """Full pages: within half a step of the code (127 steps of scale, or e4m3's half step 2^-4 of the value and
    2^-10 of the scale below its normals), the product by the inverse scale being off by 2 * 2^-24 of up to 448
    steps; unfinished pages: the very tokens."""
    c, k, v = _filled(dev, [n], 3, D, dtype, codes)
    full = n // PAGE * PAGE
    for x, h, scale in ((k, held(c, 0)[0], c.k_scale), (v, held(c, 0)[1], c.v_scale)):
        x = x[0, :, :n].double().cpu()
        assert torch.equal(h[:, full:], x[:, full:])
        if not full:
            continue
        pages = x[:, :full].reshape(3, -1, PAGE, D)
        top = pages.abs().amax((-1, -2))
        qmax = 127.0 if codes == "int8" else 448.0
        got = scale.cpu().double()[c.table[0, :full // PAGE].long().cpu()].T
        assert ((got - top / qmax).abs() <= top / qmax * 2.0 ** -22).all()
        step = (top / qmax)[..., None, None]
        err = (h[:, :full].reshape_as(pages) - pages).abs()
        if codes == "int8":
            assert (err <= step * (0.5 + 127 * 2.0 ** -21)).all()
        else:
            assert (err <= torch.maximum(pages.abs() * 2.0 ** -4, step * 2.0 ** -10) * (1 + 2.0 ** -20) + step * 2.0 ** -20).all()


@pytest.mark.parametrize("dtype,codes,D", KINDS)
def test_contents_do_not_depend_on_the_calls(dev, dtype, codes, D):
    H, T = 2, 333
    k, v = _rand((1, H, T, D), dtype, dev, 1), _rand((1, H, T, D), dtype, dev, 2)
    one = _cache(dev, H, D, 1, T, dtype, codes)
    one.append(k, v)
    for cuts in ([1] * 70 + [T - 70], [63, 1, 1, 63, 128, 77], [64, 64, 1, 63, 141], [10, 300, 23], [T - 1, 1]):
        c = _cache(dev, H, D, 1, T, dtype, codes)
        at = 0
        for m in cuts:
            c.append(k[:, :, at:at + m], v[:, :, at:at + m])
            at += m
        assert at == T and c.lengths() == [T]
        ia, ib = one.table[0, :T // PAGE].long(), c.table[0, :T // PAGE].long()
        for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
            x, y = getattr(one, name).view(torch.int8), getattr(c, name).view(torch.int8)
            assert torch.equal(x[ia], y[ib]), (name, cuts)
        for x, y in zip(held(one, 0), held(c, 0)):
            assert torch.equal(x, y)
        assert torch.equal(one.tail_top, c.tail_top)


@pytest.mark.parametrize("axes", [1, 2])
@pytest.mark.parametrize("dtype,codes,D", KINDS)
def test_rotation(dev, dtype, codes, D, axes):
    """Rotated in 32 bits (two products and a sum: 3 * 2^-24 of |x1| + |x2|) from the table's cosines and sines,
    rounded once; keys and queries alike."""
    B, H, Hq, n = 2, 2, 4, 37
    rope = RotaryTable(D, 500, base=100.0 if axes == 2 else 10000.0, axes=axes, device=dev)
    g = torch.Generator().manual_seed(5)
    pos = torch.randint(0, 500, (B, n, 2) if axes == 2 else (B, n), generator=g)
    q, k, v = _rand((B, Hq, n, D), dtype, dev, 1), _rand((B, H, n, D), dtype, dev, 2), _rand((B, H, n, D), dtype, dev, 3)
    c = _cache(dev, H, D, B, 64, dtype, codes)
    got_q = c.append(k, v, pos=pos.to(dev), rope=rope, q=q)
    d = D // axes
    inv = (100.0 if axes == 2 else 10000.0) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)

    def want(x):
        out, size = [], []
        for a, part in enumerate(x.double().cpu().split(d, -1)):
            ang = (pos[..., a] if axes == 2 else pos).double()[:, None, :, None] * inv
            x1, x2 = part[..., : d // 2], part[..., d // 2:]
            out += [x1 * ang.cos() - x2 * ang.sin(), x2 * ang.cos() + x1 * ang.sin()]
            size += [x1.abs() + x2.abs()] * 2
        return torch.cat(out, -1), torch.cat(size, -1)

    u = half_step(dtype)
    for b in range(B):
        for x, got in ((q, got_q.double().cpu()[b]), (k, held(c, b)[0])):
            w, size = want(x)
            assert ((got - w[b]).abs() <= u * w[b].abs() + (4 * 2.0 ** -24) * (1 + u) * size[b] + 1e-7).all()
        assert torch.equal(held(c, b)[1], v[b].double().cpu())
    c.check()
    # the cache of rotated keys is that of keys rotated beforehand, bit for bit
    far = _cache(dev, H, D, B, 128, dtype, codes)
    near = _cache(dev, H, D, B, 128, dtype, codes)
    kk = _rand((B, H, 128, D), dtype, dev, 9)
    pp = torch.randint(0, 500, (B, 128, 2) if axes == 2 else (B, 128), generator=g).to(dev)
    rotated = far.append(kk, kk, pos=pp, rope=rope, q=kk)
    near.append(rotated, kk)
    for b in range(B):
        for x, y in zip(held(far, b), held(near, b)):
            assert torch.equal(x, y)


def test_strides_slots_padding(dev):
    """Views of one projection at an odd offset, slots out of order, padded rows: as copies do."""
    B, H, n, D = 3, 2, 70, 64
    flat = _rand((B * n * 3 * H * D + 1,), BF16, dev, 3)
    for off in (0, 1):
        x = flat[off:off + B * n * 3 * H * D].view(B, n, 3, H, D)
        q, k, v = (x[:, :, i].transpose(1, 2) for i in range(3))
        rope = RotaryTable(D, 128, axes=2, device=dev)
        pos = torch.randint(0, 128, (B, n, 2), generator=torch.Generator().manual_seed(1)).to(dev)
        a, b = (_cache(dev, H, D, 5, 256) for _ in range(2))
        news = [70, 0, 33]
        slots = a.slots([4, 1, 2])
        qa = a.append(k, v, pos=pos, rope=rope, q=q, slots=slots, new_lens=torch.tensor(news, dtype=torch.int32, device=dev))
        for i, s in enumerate([4, 1, 2]):
            m = news[i]
            qb = b.append(k[i:i + 1, :, :m].contiguous(), v[i:i + 1, :, :m].contiguous(), pos=pos[i:i + 1, :m], rope=rope,
                          q=q[i:i + 1, :, :m].contiguous(), slots=[s])
            assert torch.equal(qa[i:i + 1, :, :m], qb)
            assert (qa[i, :, m:] == 0).all()
        assert a.lengths() == b.lengths() == [0, news[1], news[2], 0, news[0]]
        for s in range(5):
            for x, y in zip(held(a, s), held(b, s)):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,codes,D", KINDS)
def test_read(dev, dtype, codes, D):
    lens = [0, 5, 64, 200]
    c, _, _ = _filled(dev, lens, 2, D, dtype, codes)
    for n, start in ((70, None), (130, [0, -3, 64, 66]), (1, [0, 4, 63, 199])):
        st = None if start is None else torch.tensor(start, dtype=torch.int32, device=dev)
        k, v = c.read(n, start=st)
        for b, L in enumerate(lens):
            s = L - n if start is None else start[b]
            for got, x in zip((k, v), held(c, b)):
                want = torch.zeros(2, n, D, dtype=torch.float64)
                lo, hi = max(s, 0), min(max(s + n, 0), L)
                if hi > lo:
                    want[:, lo - s:hi - s] = x[:, lo:hi]
                assert ((got[b].double().cpu() - want).abs() <= half_step(dtype) * want.abs() * (1 + 2.0 ** -10)
                        + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()


# ---- attention --------------------------------------------------------------
def _check(c, q, got, n_new=None, causal=False, scale=None, slots=None):
    B, n = q.shape[0], q.shape[2]
    for b in range(B):
        s = b if slots is None else slots[b]
        m = n if n_new is None else n_new[b]
        k, v = held(c, s)
        want, size, spread = attention(q[b], k, v, m, causal, scale)
        err = (got[b].double().cpu() - want).abs()
        tol = tolerance(want, size, spread, q.dtype, k.shape[1])
        assert torch.isfinite(got[b]).all()
        assert (err <= tol).all(), (b, float((err / tol).max()))


@pytest.mark.parametrize("dtype,codes,D", KINDS)
@pytest.mark.parametrize("n,G", [(1, 1), (1, 4), (3, 2), (17, 1), (33, 1), (40, 4), (130, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_attend(dev, dtype, codes, D, n, G, causal):
    lens = [max(n, L) for L in (1, 63, 64, 65, 300)]
    c, _, _ = _filled(dev, lens, 2, D, dtype, codes)
    q = _rand((len(lens), 2 * G, n, D), dtype, dev, 7, 1.5)
    _check(c, q, c.attend(q, causal=causal), causal=causal)


@pytest.mark.parametrize("dtype,codes,D", KINDS)
@pytest.mark.parametrize("n,L", [(1, 9000), (5, 4097), (64, 5000), (257, 3333)])
def test_attend_split(dev, dtype, codes, D, n, L):
    """Long caches, whose keys are split over workgroups and joined."""
    c, _, _ = _filled(dev, [L, L // 3], 1, D, dtype, codes)
    q = _rand((2, 1, n, D), dtype, dev, 7, 1.5)
    for causal in (False, True):
        _check(c, q, c.attend(q, causal=causal), causal=causal)


@pytest.mark.parametrize("dtype,codes", [(BF16, "int8"), (BF16, "fp8"), (F16, "int8"), (F16, "fp8")])
@pytest.mark.parametrize("n,G", [(129, 1), (256, 1), (60, 4), (250, 2)])
def test_attend_wide_tiles(dev, dtype, codes, n, G):
    """Workgroups of eight waves, over ragged caches: the longest in parts, others in one, one shorter than its rows."""
    lens = [5000, 4100, 700, n // 2]
    c, _, _ = _filled(dev, lens, 1, 64, dtype, codes)
    q = _rand((len(lens), G, n, 64), dtype, dev, 7, 1.5)
    for causal in (False, True):
        _check(c, q, c.attend(q, causal=causal), causal=causal)
    news = [n, n - 100 if n > 100 else 1, 0, n // 2]
    _check(c, q, c.attend(q, causal=True, new_lens=news), n_new=news, causal=True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [5, 200])
def test_attend_parts_not_finite(dev, D, n):
    """A page that is not finite in the second part of a split cache: its rows are NaN, other sequences' as before, and
    so are the rows of a causal chunk that end before it."""
    T = 9000
    c, k, v = _filled(dev, [T, T], 1, D)
    q = _rand((2, 1, n, D), BF16, dev, 3)
    want = c.attend(q, causal=True)
    at = T - n // 2
    for name in ("k", "v"):
        d, _, _ = _filled(dev, [at, T], 1, D)
        kk, vv = k[:, :, at:].clone(), v[:, :, at:].clone()
        (kk if name == "k" else vv)[0, 0, 0, 3] = float("nan")
        d.append(kk[:1], vv[:1], slots=[0])
        got = d.attend(q, causal=True)
        assert torch.equal(got[1], want[1])
        hit = max(0, at // PAGE * PAGE - (T - n))
        assert torch.isfinite(got[0, 0, :hit]).all() and got[0, 0, n - n // 2:].isnan().all()
        assert torch.equal(got[0, 0, :hit], want[0, 0, :hit])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n", [8, 48])
def test_attend_rows_that_see_nothing(dev, dtype, n):
    """Empty sequences and causal rows ahead of the first token give zeros; padding of a given out stays."""
    c, _, _ = _filled(dev, [0, 3, 100], 2, 64, dtype)
    q = _rand((3, 4, n, 64), dtype, dev, 5)
    got = c.attend(q, causal=True)
    _check(c, q, got, causal=True)
    assert (got[0] == 0).all() and (got[1, :, : n - 3] == 0).all()
    assert (c.attend(q)[0] == 0).all()
    news = [n, 2, n - 3]
    out = torch.full_like(q, 7.0)
    got = c.attend(q, new_lens=news, out=out)
    assert got is out
    for b, m in enumerate(news):
        assert (out[b, :, m:] == 7.0).all()
    fresh = c.attend(q, new_lens=torch.tensor(news, dtype=torch.int32, device=dev))
    _check(c, q, fresh, n_new=news)
    for b, m in enumerate(news):
        assert torch.equal(fresh[b, :, :m], out[b, :, :m]) and (fresh[b, :, m:] == 0).all()


def test_attend_strides_and_slots(dev):
    c, _, _ = _filled(dev, [70, 200, 10], 2)
    for off in (0, 1):
        flat = _rand((2 * 20 * 4 * 64 + 1,), BF16, dev, 4)
        q = flat[off:off + 2 * 20 * 4 * 64].view(2, 20, 4, 64).transpose(1, 2)
        store = torch.zeros(2 * 20 * 4 * 64 + 1, dtype=BF16, device=dev)
        out = store[off:off + 2 * 20 * 4 * 64].view(2, 20, 4, 64).transpose(1, 2)
        c.attend(q, slots=[2, 1], out=out)
        _check(c, q, out, slots=[2, 1])
        assert torch.equal(out, c.attend(q.contiguous(), slots=[2, 1]))


@pytest.mark.parametrize("dtype,codes,D", KINDS)
def test_attend_ranges(dev, dtype, codes, D):
    """Values from tiny to the type's largest, pages of zeros, and one key that takes all the weight."""
    H, T = 1, 200
    big = 3.0e4 if dtype == F16 else 1e30
    for gain in (1e-4, big):
        c = _cache(dev, H, D, 1, T, dtype, codes)
        k, v = _rand((1, H, T, D), dtype, dev, 1), (_rand((1, H, T, D), torch.float32, dev, 2).clamp(-2, 2) * gain).to(dtype)
        v[:, :, 64:128] = 0
        k[:, :, :64] = 0
        c.append(k, v)
        q = _rand((1, H, 5, D), dtype, dev, 3)
        _check(c, q, c.attend(q))
        qq = q.expand(1, H, 5, D).repeat(1, 1, 10, 1)
        _check(c, qq, c.attend(qq))
    # a v_scale that falls and rises by orders of magnitude from page to page
    c = _cache(dev, H, D, 1, 512, dtype, codes)
    v = _rand((1, H, 500, D), torch.float32, dev, 2).clamp(-2, 2)
    v = (v * (10.0 ** torch.tensor([-3, 2, -2, 4, 0, -1, 3, 1], device=dev)).repeat_interleave(64)[:500, None]).to(dtype)
    c.append(_rand((1, H, 500, D), dtype, dev, 1), v)
    for n in (3, 70):
        q = _rand((1, H, n, D), dtype, dev, 3)
        _check(c, q, c.attend(q))
    # scores hundreds apart
    k = _rand((1, H, 500, D), dtype, dev, 11, 8.0)
    c = _cache(dev, H, D, 1, 512, dtype, codes)
    c.append(k, _rand((1, H, 500, D), dtype, dev, 2))
    for n in (3, 70):
        q = _rand((1, H, n, D), dtype, dev, 3, 8.0)
        _check(c, q, c.attend(q))


@pytest.mark.parametrize("dtype,codes,D", KINDS)
@pytest.mark.parametrize("n,T", [(3, 100), (3, 5000), (100, 700), (100, 5000)])
def test_attend_largest_values(dev, dtype, codes, D, n, T):
    """Values at the type's largest under weights that are all alike: no sum of them is formed, whole or in parts."""
    top = torch.finfo(dtype).max
    c = _cache(dev, 1, D, 1, T, dtype, codes)
    k = torch.zeros(1, 1, T, D, dtype=dtype, device=dev)
    v = torch.full((1, 1, T, D), top, dtype=dtype, device=dev)
    v[..., 1::2] *= -1
    c.append(k, v)
    got = c.attend(torch.ones(1, 1, n, D, dtype=dtype, device=dev)).double()
    want = v[:, :, :n].double()
    assert torch.isfinite(got).all() and ((got - want).abs() <= top * 3 * half_step(dtype)).all()


@pytest.mark.parametrize("dtype,codes,D", KINDS)
@pytest.mark.parametrize("n", [20, 100])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("at", [100, 150])
def test_values_that_are_not_finite(dev, dtype, codes, D, n, which, at):
    """A NaN or infinity, in a full page (token 100) or the unfinished one (150), reaches the rows that see its
    page (a full one) or its token (the unfinished one) and no others: not earlier rows of a causal chunk, not
    other heads, not other sequences."""
    T = 160
    k, v = _rand((2, 2, T, D), dtype, dev, 1), _rand((2, 2, T, D), dtype, dev, 2)
    clean = _cache(dev, 2, D, 2, T, dtype, codes)
    clean.append(k, v)
    q = _rand((2, 2, n, D), dtype, dev, 3)
    want = clean.attend(q, causal=True)
    clean.check()
    for bad in (float("nan"), float("inf")):
        kk, vv = k.clone(), v.clone()
        (kk if which == "k" else vv)[1, 0, at, 3] = bad
        c = _cache(dev, 2, D, 2, T, dtype, codes)
        c.append(kk, vv)
        got = c.attend(q, causal=True)
        lo = T - n
        page = at // PAGE * PAGE if at < 128 or which == "v" else at
        hit = max(0, page - lo)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1, 1], want[1, 1])
        assert torch.equal(got[1, 0, :hit], want[1, 0, :hit])
        if at < 128 or which == "v" or math.isnan(bad):
            assert got[1, 0, hit:].isnan().all()
        if at < 128:
            with pytest.raises(RuntimeError, match="not finite"):
                c.check()
        c.check()


# ---- the cache's life -------------------------------------------------------
def test_snapshot_restore_release(dev):
    c, k, v = _filled(dev, [70, 130], 2)
    before = [held(c, s) for s in range(2)]
    snap = c.snapshot()
    more = _rand((2, 2, 100, 64), BF16, dev, 9)
    c.append(more[:, :, :60], more[:, :, :60])
    later = c.snapshot()
    c.restore(snap)
    assert c.lengths() == [70, 130]
    for s in range(2):
        for x, y in zip(before[s], held(c, s)):
            assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="no longer holds"):
        c.restore(later)
    c.append(more[:, :, :10], more[:, :, :10])
    q = _rand((2, 2, 10, 64), BF16, dev, 1)
    _check(c, q, c.attend(q, causal=True), causal=True)
    free = c.free_pages()
    c.release(1)
    assert c.free_pages() == free + 3 and c.lengths() == [80, 0]
    with pytest.raises(RuntimeError, match="no longer holds"):
        c.restore(snap)
    c.append(more[:1], more[:1], slots=[1])
    assert c.lengths() == [80, 100]
    for s, L in ((0, 80), (1, 100)):
        _check(c, q[:1], c.attend(q[:1], slots=[s], causal=True), causal=True, slots=[s])


def test_pages_run_out(dev):
    c = PagedKVCache(4, 1, 64, max_seqs=2, max_len=192, device=dev)
    x = _rand((2, 1, 200, 64), BF16, dev, 0)
    with pytest.raises(ValueError, match="max_len"):
        c.append(x[:1], x[:1])
    c.append(x[:1, :, :150], x[:1, :, :150])
    with pytest.raises(RuntimeError, match="free pages"):
        c.append(x[1:, :, :130], x[1:, :, :130], slots=[1])
    assert c.lengths() == [150, 0] and c.free_pages() == 1
    # a padded batch that is estimated too long is measured before it is refused
    one = torch.tensor([1], dtype=torch.int32, device=dev)
    for _ in range(5):
        c.append(x[:1, :, :40], x[:1, :, :40], new_lens=one)
    assert c.lengths()[0] == 155
    c.append(x[1:, :, :64], x[1:, :, :64], slots=[1])
    q = _rand((2, 1, 1, 64), BF16, dev, 1)
    _check(c, q, c.attend(q))
    # tokens past the reserved pages are dropped and reported (the host's estimate made wrong on purpose)
    c._bound[0] = 0
    c.append(x[:1, :, :60], x[:1, :, :60])
    assert c.lengths()[0] == 192
    with pytest.raises(RuntimeError, match="dropped"):
        c.check()
    _check(c, q, c.attend(q))


def test_padding_takes_no_pages(dev):
    """Counts that the host does not see: a sequence that gets no tokens takes no further pages, calls on end."""
    c = PagedKVCache(6, 1, 64, max_seqs=2, device=dev)
    x = _rand((2, 1, 64, 64), BF16, dev, 0)
    news = torch.tensor([64, 0], dtype=torch.int32, device=dev)
    for _ in range(5):
        c.append(x, x, new_lens=news)
    assert c.lengths() == [320, 0] and c.free_pages() == 0
    c.check()


def test_captured_restore(dev):
    """A restore recorded in a graph has not run: the host's bounds are not taken for the lengths after it."""
    c = _cache(dev, 1, 64, 1, 64 * 6)
    x = _rand((1, 1, 150, 64), BF16, dev, 0)
    c.append(x[:, :, :100], x[:, :, :100])
    snap = c.snapshot()
    c.append(x, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.restore(snap)
    c.append(x[:, :, :100], x[:, :, :100])
    assert c.lengths() == [350]
    for m in (100, 30):
        graph.replay()
        torch.cuda.synchronize()
        c.append(x[:, :, :m], x[:, :, :m])
        assert c.lengths() == [100 + m]
        q = x[:, :, :2].contiguous()
        _check(c, q, c.attend(q))
    c.check()
    with pytest.raises(RuntimeError, match="not inside a graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            c.release(0)


def test_positions_outside_the_table(dev):
    c = _cache(dev)
    rope = RotaryTable(64, 10, axes=1, device=dev)
    x = _rand((1, 2, 3, 64), BF16, dev, 0)
    a = c.append(x, x, pos=torch.tensor([[0, 10, -1]], device=dev), rope=rope, q=x)
    with pytest.raises(RuntimeError, match="rotation table"):
        c.check()
    b = c.append(x, x, pos=torch.tensor([[0, 9, 0]], device=dev), rope=rope, q=x)
    c.check()
    assert torch.equal(a, b)


def test_page_numbers_outside_the_pool(dev):
    """A table changed from outside: such a page is neither read nor written, and is reported."""
    c, _, _ = _filled(dev, [200], 2)
    q = _rand((1, 2, 3, 64), BF16, dev, 1)
    good = c.table.clone()
    for n in (3, 50):
        qq = _rand((1, 2, n, 64), BF16, dev, 1)
        c.table[0, 1] = c.n_pages + 5
        assert torch.isfinite(c.attend(qq)).all()
        with pytest.raises(RuntimeError, match="pool"):
            c.check()
        c.table.copy_(good)
    c.table[0, 3] = -7
    x = _rand((1, 2, 60, 64), BF16, dev, 2)
    c.append(x, x)
    with pytest.raises(RuntimeError, match="pool"):
        c.check()
    c.read(10)
    c.table.copy_(good)
    assert torch.isfinite(c.attend(q)).all()


def test_far_pages(dev):
    """Pages whose codes lie past 2^31 bytes."""
    H, D = 16, 128
    per = H * PAGE * D
    n_pages = (1 << 31) // per + 40
    c = PagedKVCache(n_pages, H, D, max_seqs=2, device=dev)
    c.reserve(0, PAGE * (n_pages - 5))
    x = _rand((1, H, 200, D), BF16, dev, 2)
    c.append(x, x, slots=[1])
    assert int(c.table[1, :3].min()) * per > 1 << 31
    near = _cache(dev, H, D, 1, 256)
    near.append(x, x)
    for n in (2, 60):
        q = _rand((1, H, n, D), BF16, dev, 3)
        assert torch.equal(c.attend(q, slots=[1]), near.attend(q))
    for a, b in zip(c.read(200, slots=[1]), near.read(200)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [1, 40])
def test_captured_steps(dev, n):
    """append and attend captured in one graph and replayed: each replay appends, as the same eager calls do."""
    B, H, D, steps = 2, 2, 64, 5
    eager, c = (_filled(dev, [50, 61], H, D, room=steps * n + 64)[0] for _ in range(2))
    xs = [_rand((B, H, n, D), BF16, dev, 20 + i) for i in range(steps)]
    rope = RotaryTable(D, 64, axes=2, device=dev)
    ps = [torch.randint(0, 64, (B, n, 2), generator=torch.Generator().manual_seed(i)).to(dev) for i in range(steps)]
    want = []
    for x, p in zip(xs, ps):
        want.append(eager.attend(eager.append(x, x, pos=p, rope=rope, q=x), causal=True))
    for s in range(B):
        c.reserve(s, 61 + steps * n)
    x, p = xs[0].clone(), ps[0].clone()
    snap = c.snapshot()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attend(c.append(x, x, pos=p, rope=rope, q=x), causal=True)
    torch.cuda.current_stream().wait_stream(side)
    c.restore(snap)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attend(c.append(x, x, pos=p, rope=rope, q=x), causal=True)
    for i in range(steps):
        x.copy_(xs[i])
        p.copy_(ps[i])
        graph.replay()
        torch.cuda.synchronize()
        err = (out.double() - want[i].double()).abs().max()
        assert err <= 2 * half_step(BF16) * want[i].double().abs().max(), i
        assert torch.equal(c.lens, torch.tensor([50 + (i + 1) * n, 61 + (i + 1) * n], dtype=torch.int32, device=dev))
    for s in range(B):
        for a, b in zip(held(eager, s), held(c, s)):
            assert torch.equal(a, b)
    # eager calls after the replays know the lengths
    y = _rand((B, H, 3, D), BF16, dev, 77)
    c.append(y, y)
    c.check()
    assert c.lengths() == [53 + steps * n, 64 + steps * n]
    with pytest.raises(RuntimeError, match="made before it"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            c.append(y, y, new_lens=[3, 3])
    with pytest.raises(RuntimeError, match="made before it"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            c.attend(y, slots=[0, 1])
    full = _cache(dev, H, D, 1, 64)
    with pytest.raises(RuntimeError, match="reserved before"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            full.append(y[:1], y[:1])


def test_another_stream(dev):
    c, _, _ = _filled(dev, [300], 2)
    q = _rand((1, 2, 7, 64), BF16, dev, 1)
    want = c.attend(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.attend(q)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(dev):
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVCache(4, 2, 80, device=dev)
    with pytest.raises(TypeError, match="dtype"):
        PagedKVCache(4, 2, dtype=torch.float32, device=dev)
    with pytest.raises(ValueError, match="codes"):
        PagedKVCache(4, 2, codes="int4", device=dev)
    with pytest.raises(ValueError, match="at least 1"):
        PagedKVCache(0, 2, device=dev)
    with pytest.raises(ValueError, match="max_len"):
        PagedKVCache(4, 2, max_len=0, device=dev)
    many = torch.zeros(1, 1, 1, 64, dtype=BF16, device=dev).expand(1, 1, (1 << 30) + 1, 64)
    one = PagedKVCache(4, 1, device=dev)
    with pytest.raises(ValueError, match="rows"):
        one.append(many, many, new_lens=torch.ones(1, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="rows"):
        one.attend(many)
    c, _, _ = _filled(dev, [70], 2)
    x = _rand((1, 2, 5, 64), BF16, dev, 0)
    rope = RotaryTable(64, 16, axes=2, device=dev)
    pos = torch.zeros(1, 5, 2, dtype=torch.int64, device=dev)
    for bad, err in ((x.cpu(), RuntimeError), (x.float(), TypeError), (x[..., :32], ValueError), (x[0], ValueError),
                     (x[:, :1], ValueError), (x.repeat(1, 1, 1, 2)[..., ::2], ValueError),
                     (x.repeat(2, 1, 1, 1), ValueError)):
        with pytest.raises(err):
            c.append(bad, bad)
    with pytest.raises(ValueError, match="batch and tokens"):
        c.append(x, x[:, :, :4])
    with pytest.raises(ValueError, match="go together"):
        c.append(x, x, pos=pos)
    with pytest.raises(ValueError, match="needs pos"):
        c.append(x, x, q=x)
    for bad in (pos[:, :, 0], pos.float(), pos[:, :4]):
        with pytest.raises(ValueError, match="pos must"):
            c.append(x, x, pos=bad, rope=rope)
    with pytest.raises(ValueError, match="rope is for"):
        c.append(x, x, pos=pos, rope=RotaryTable(128, 16, axes=2, device=dev))
    for bad in ([1, 2], [6], torch.tensor([1], device=dev), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(ValueError, match="new_lens"):
            c.append(x, x, new_lens=bad)
    with pytest.raises(ValueError, match="once"):
        _cache(dev, S=3).append(x.repeat(2, 1, 1, 1), x.repeat(2, 1, 1, 1), slots=[1, 1])
    with pytest.raises(IndexError):
        c.append(x, x, slots=[1])
    with pytest.raises(ValueError, match="multiple of 2"):
        c.attend(_rand((1, 3, 5, 64), BF16, dev, 0))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            c.attend(x, scale=scale)
    with pytest.raises(ValueError, match="out must"):
        c.attend(x, out=x[:, :, :4])
    with pytest.raises(ValueError, match="expanded"):
        c.attend(x, out=x[:, :1].expand(1, 2, 5, 64))
    with pytest.raises(RuntimeError, match="no backward"):
        c.attend(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="start"):
        c.read(3, start=torch.zeros(1, device=dev))
    assert c.lengths() == [70]
    for empty in (x[:, :, :0], x[:0]):
        assert c.attend(empty).shape == empty.shape
        assert c.append(empty, empty) is None
