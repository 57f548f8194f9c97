"""Attention and its gradients in 64 bits with the roundings that the kernels make (P, dS, each result), for tests that hold an error's
norm to that of the same roundings: worst-case bounds of every element add up errors of one sign, and see a few percent of a
gradient go wrong only where it is far above them."""

import math

import torch

BITS = {torch.bfloat16: 8, torch.float16: 11}


def rounded(x, dt):
    """x (64 bits) to the type's bits, without its range."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 2.0 ** BITS[dt]) * 2.0 ** -BITS[dt], e)


def attention(q, k, v, see, do, dt=None):
    """[out, dq, dk, dv] in 64 bits; with dt, of operands and with intermediate values rounded to it."""
    r = (lambda x: x) if dt is None else (lambda x: rounded(x, dt))
    B, Hq, Tq, D = q.shape
    Hk, Tk = k.shape[1], k.shape[2]
    scale, see = 1.0 / math.sqrt(D), see.to(q.device)
    q, g = (torch.where(see.any(3)[..., None], t.detach().double(), 0.0) for t in (q, do))
    kr, vr = (t.detach().double().repeat_interleave(Hq // Hk, 1) for t in (k, v))
    used = see.any(2)[..., None]
    kr, vr = torch.where(used, kr, 0.0), torch.where(used, vr, 0.0)
    s = (q @ kr.transpose(2, 3).contiguous() * scale).masked_fill(~see, -math.inf)
    e = torch.where(see, (s - s.amax(-1, keepdim=True)).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    over = torch.where(total > 0, 1.0 / total, 0.0)
    o = r(e) @ vr * over
    p = e * over
    ds = r(p * (g @ vr.transpose(2, 3).contiguous() - (g * o).sum(-1, keepdim=True)))

    def back(x):
        return x.reshape(B, Hk, Hq // Hk, Tk, D).sum(2)

    return [r(o), r(scale * (ds @ kr)), r(back(scale * (ds.transpose(2, 3).contiguous() @ q))),
            r(back(r(p).transpose(2, 3).contiguous() @ g))]


def off(x, want):
    """The error's norm relative to the values'."""
    return ((x.double() - want).norm() / want.norm()).item()
