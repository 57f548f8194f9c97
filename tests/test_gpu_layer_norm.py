"""ress_amd.layer_norm, ress_amd.add_layer_norm and their gradients against the definition in 64 bits. Tolerances: half a step of the
result's type (eps / 2 relative), and 2^-18 of the magnitudes that a 32-bit sum or difference goes through (a row or a
column of up to 2^6 sums of 2^-24 each, taken a piece after the other)."""

import pytest
import torch

import ress_amd as ress

pytestmark = pytest.mark.gpu
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
SLACK = 2.0 ** -18


def make(shape, dt, wt, seed=0, affine=True, branch=False, gamma=False, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]

    def one(*s, by=1.0, plus=0.0, t=dt):
        return (torch.randn(*s, generator=g) * by + plus).to(t).cuda().requires_grad_()

    x = one(*shape, plus=offset)
    return {"x": x, "branch": one(*shape, by=0.7) if branch else None, "gamma": one(C, by=0.3, plus=0.5, t=wt) if gamma else None,
            "weight": one(C, by=0.2, plus=1.0, t=wt) if affine else None, "bias": one(C, by=0.1, t=wt) if affine else None,
            "dh": one(*shape, by=0.1).detach() if branch else None, "dn": one(*shape, by=0.1).detach()}


def run(s, eps=1e-5):
    if s["branch"] is None:
        outs = (ress.layer_norm(s["x"], s["weight"], s["bias"], eps),)
        grads = (s["dn"],)
    else:
        outs = ress.add_layer_norm(s["x"], s["branch"], s["gamma"], s["weight"], s["bias"], eps)
        grads = (s["dh"], s["dn"])
    names = [n for n in ("x", "branch", "gamma", "weight", "bias") if s[n] is not None]
    got = torch.autograd.grad(outs, [s[n] for n in names], grads)
    return dict(zip(("n",) if s["branch"] is None else ("h", "n"), outs), **dict(zip(names, got)))


def check(s, eps=1e-5):
    got = run(s, eps)
    dt = s["x"].dtype
    C = s["x"].shape[-1]
    x = s["x"].detach().double()
    one = torch.ones(C, dtype=torch.float64, device=x.device)
    w = one if s["weight"] is None else s["weight"].detach().double()
    b = 0 * one if s["bias"] is None else s["bias"].detach().double()
    gamma = one if s["gamma"] is None else s["gamma"].detach().double()
    u, tiny = STEP[dt], TINY[dt]

    def near(name, value, bound):
        t = got[name]
        assert torch.isfinite(t).all(), name
        bound = bound + STEP[t.dtype] * value.abs() + TINY[t.dtype]
        off = (t.double() - value).abs()
        assert (off <= bound).all(), f"{name}: {(off / bound.clamp(min=1e-300)).max().item():.2f} of the bound"

    h = x
    if s["branch"] is not None:
        br = s["branch"].detach().double()
        near("h", x + gamma * br, SLACK * (x.abs() + (gamma * br).abs()))
        h = got["h"].detach().double()  # the norm is that of the sum as returned
    mean = h.mean(-1, keepdim=True)
    rstd = ((h - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (h - mean) * rstd
    fuzz = SLACK * (h.abs().amax(-1, keepdim=True) * rstd + xh.abs()) * (1 + xh.abs())  # of xh, through mean and rstd
    near("n", xh * w + b, fuzz * w.abs() + SLACK * b.abs())
    dn = s["dn"].double()
    g = dn * w
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    err = rstd * (SLACK * (g.abs() + g.abs().mean(-1, keepdim=True) + (xh * c2).abs())
                  + fuzz * c2.abs() + xh.abs() * (SLACK * (g * xh).abs().mean(-1, keepdim=True) + (g.abs() * fuzz).mean(-1, keepdim=True)))
    err = err + SLACK * dx.abs() + fuzz * dx.abs()
    if s["dh"] is not None:
        dx = dx + s["dh"].double()
        err = err + SLACK * s["dh"].double().abs()
    near("x", dx, err)
    lead = tuple(range(x.dim() - 1))
    if s["branch"] is not None:
        near("branch", gamma * dx, gamma.abs() * err)
        if s["gamma"] is not None:
            near("gamma", (dx * br).sum(lead), (err * br.abs() + SLACK * (dx * br).abs()).sum(lead))
    if s["weight"] is not None:
        near("weight", (dn * xh).sum(lead), (dn.abs() * fuzz + SLACK * (dn * xh).abs()).sum(lead))
        near("bias", dn.sum(lead), SLACK * dn.abs().sum(lead))
    return got


WIDTHS = [1, 2, 7, 8, 33, 63, 64, 65, 72, 128, 136, 384, 511, 512, 520, 1000, 1023, 1024, 1032, 2048, 2056, 2500, 4096, 4100, 5000, 8191, 8192]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("C", WIDTHS)
def test_widths(dev, dt, C):
    check(make((5, C), dt, dt))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("C", [7, 64, 100, 1024, 2048, 3000, 8192])
@pytest.mark.parametrize("gamma", [False, True])
def test_residual_sums(dev, dt, C, gamma):
    check(make((3, 11, C), dt, dt, branch=True, gamma=gamma))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [64, 77, 1024, 2048])
@pytest.mark.parametrize("rows", [1, 2, 63, 513, 5000])
def test_rows_and_weights_in_32_bits(dev, dt, C, rows):
    check(make((rows, C), dt, torch.float32, branch=C != 64, gamma=C == 1024))


def test_many_rows(dev):
    """More rows than a launch has workgroups' worth, of the smallest width."""
    check(make((200_001, 8), torch.bfloat16, torch.float32))


@pytest.mark.parametrize("branch", [False, True])
def test_no_weights(dev, branch):
    check(make((9, 96), torch.bfloat16, torch.bfloat16, affine=False, branch=branch))


def test_only_some_weights(dev):
    x, w = torch.randn(6, 64, device=dev), torch.randn(64, device=dev)
    assert torch.equal(ress.layer_norm(x, w), ress.layer_norm(x, w, torch.zeros(64, device=dev)))
    assert torch.equal(ress.layer_norm(x, None, w), ress.layer_norm(x, torch.ones(64, device=dev), w))


@pytest.mark.parametrize("C", [64, 1024])
def test_rows_far_from_zero(dev, C):
    """A mean a thousand times the deviation: the variance is taken of the differences."""
    s = make((40, C), torch.float32, torch.float32, offset=1000.0)
    check(s)


def test_a_constant_row(dev):
    x = torch.full((3, 100), 7.0, device=dev, requires_grad=True)
    n = ress.layer_norm(x)
    assert (n == 0).all()
    g, = torch.autograd.grad(n, x, torch.randn(3, 100, device=dev))
    assert torch.isfinite(g).all()


@pytest.mark.parametrize("C", [64, 128, 100])
def test_rows_read_in_place(dev, C):
    """Heads of a projection's output, transposed, expanded and unaligned rows: the contiguous call's bits."""
    g = torch.Generator().manual_seed(0)
    w, b = (torch.randn(C, generator=g).cuda().bfloat16().requires_grad_() for _ in range(2))
    y = torch.randn(2, 30, 3, 4, C, generator=g).cuda().bfloat16()
    dn = torch.randn(2, 4, 30, C, generator=g).cuda().bfloat16()
    views = [y.permute(2, 0, 3, 1, 4)[1], y[:, :, 0].transpose(1, 2), y[:1, :, 2].transpose(1, 2).expand(2, -1, -1, -1)]
    views.append(torch.zeros(2, 4, 30, C + 3, device=dev).bfloat16()[..., 3:].copy_(views[0]))
    views.append(y.unsqueeze(0).permute(3, 0, 1, 4, 2, 5)[1].squeeze(0))
    for v in views:
        x1, x2 = v.detach().requires_grad_(), v.detach().contiguous().requires_grad_()
        outs = []
        for x in (x1, x2):
            n = ress.layer_norm(x, w, b)
            outs.append((n, *torch.autograd.grad(n, (x, w, b), dn if x is x2 else dn.transpose(1, 2).contiguous().transpose(1, 2))))
        assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_only_one_result_is_used(dev):
    """The other's gradient is zero."""
    s = make((7, 200), torch.bfloat16, torch.bfloat16, branch=True, gamma=True)
    names = ("x", "branch", "gamma", "weight", "bias")
    leaves = [s[n] for n in names]
    zero = torch.zeros_like(s["dn"])
    h, n = ress.add_layer_norm(*leaves)
    only_n = torch.autograd.grad(n, leaves, s["dn"], retain_graph=True)
    both = torch.autograd.grad((h, n), leaves, (zero, s["dn"]), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(only_n, both))
    only_h = torch.autograd.grad(h, leaves, s["dh"], allow_unused=True)
    assert torch.equal(only_h[0], s["dh"])
    assert all(t is None or (t == 0).all() for t in only_h[3:])
    frozen = ress.add_layer_norm(s["x"], s["branch"].detach(), s["gamma"].detach(), s["weight"].detach(), s["bias"].detach())
    assert torch.equal(torch.autograd.grad(frozen, s["x"], (zero, s["dn"]))[0], only_n[0])


def test_empty(dev):
    for shape in ((0, 64), (3, 0, 64)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        w = torch.ones(64, device=dev, requires_grad=True)
        n = ress.layer_norm(x, w)
        gx, gw = torch.autograd.grad(n, (x, w), torch.zeros(shape, device=dev))
        assert n.shape == gx.shape == x.shape and (gw == 0).all()


def test_repeats_and_another_stream(dev):
    s = make((3000, 1024), torch.bfloat16, torch.float32, branch=True, gamma=True)
    first = run(s)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        second = run(s)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(first[n], second[n]) for n in first)


def test_captured(dev):
    s = make((70, 1024), torch.bfloat16, torch.bfloat16, branch=True, gamma=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(s)
    for i in range(4):
        new = make((70, 1024), torch.bfloat16, torch.bfloat16, branch=True, gamma=True, seed=i + 1)
        with torch.no_grad():
            for n in s:
                s[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        want = run(new)
        assert all(torch.equal(got[n], want[n]) for n in want), i


def test_against_differences(dev):
    """The directional derivative of sum(n * dn) by differences of the definition in 64 bits."""
    s = make((4, 50), torch.float32, torch.float32)
    got = run(s)
    g = torch.Generator().manual_seed(5)

    def value(x, w, b):
        c = x - x.mean(-1, keepdim=True)
        return ((c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b) * s["dn"].double()).sum()

    at = {n: s[n].detach().double() for n in ("x", "weight", "bias")}
    for n in at:
        d = torch.randn(at[n].shape, generator=g).to(dev).double()
        h = 1e-5
        diff = (value(*[t + h * d if m == n else t for m, t in at.items()])
                - value(*[t - h * d if m == n else t for m, t in at.items()])) / (2 * h)
        # fp32 gradients: 2^-18 of the terms; differences: h^2 and 2^-52 / h of the value's terms
        bound = SLACK * (got[n].double() * d).abs().sum() * 8 + 1e-6
        assert ((got[n].double() * d).sum() - diff).abs() <= bound


def test_offsets_past_32_bits(dev):
    """Four million rows of 1,024: the last ones as a call of their own."""
    few = make((64, 1024), torch.bfloat16, torch.bfloat16, branch=True, gamma=True)
    few = {n: None if t is None else t.detach() for n, t in few.items()}
    many = {n: t.repeat(65537, 1) if t.dim() == 2 else t for n, t in few.items()}
    a, b = ({n: t.requires_grad_() if n[0] != "d" else t for n, t in s.items()} for s in (few, many))
    want, got = run(a), run(b)
    for n in ("h", "n", "x", "branch"):
        assert torch.equal(got[n][:64], want[n]) and torch.equal(got[n][-64:], want[n]), n
