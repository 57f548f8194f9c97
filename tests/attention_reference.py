"""Attention and its gradients in 64 bits from the definition, with bounds on what 16-bit operands and results may be off
by: the reference of the tests of ress_amd.block_attention."""

import math

import torch

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # a rounding is off by at most half a step: eps / 2


def visible(B, Hq, Tq, Tk, causal=False, q_lens=None, k_lens=None, block_map=None):
    """(B, Hq, Tq, Tk) bool: what a row sees."""
    ql = [Tq] * B if q_lens is None else q_lens
    kl = [Tk] * B if k_lens is None else k_lens
    see = torch.zeros(B, Hq, Tq, Tk, dtype=torch.bool)
    i, j = torch.arange(Tq)[:, None], torch.arange(Tk)[None]
    for b in range(B):
        s = (i < ql[b]) & (j < kl[b])
        if causal:
            s = s & (j <= i + kl[b] - ql[b])
        see[b] = s
    if block_map is not None:
        m = block_map.cpu().bool().expand(B, Hq, -1, -1)
        see &= m.repeat_interleave(128, 2)[:, :, :Tq].repeat_interleave(64, 3)[..., :Tk]
    return see


def reference(q, k, v, see, scale=None, grad=None):
    """{name: (value, bound)} of out, and with grad of dq, dk, dv, in 64 bits on the operands' device. The bounds count half a step
    for each rounding to the operands' type (P, dS and the result; delta carries P's), fp16's smallest step where a
    value lies below its range, and 2^-16 of the sums of magnitudes for everything in 32 bits."""
    dt, dev = q.dtype, q.device
    B, Hq, Tq, D = q.shape
    Hk, Tk = k.shape[1], k.shape[2]
    G = Hq // Hk
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    see = see.to(dev)
    u, tiny = STEP[dt], 2.0 ** -25 if dt is torch.float16 else 0.0
    q64, k64, v64 = (t.detach().double() for t in (q, k, v))
    k64, v64 = (torch.where(see.any(2).reshape(B, Hk, G, Tk).any(2)[..., None], t, 0.0) for t in (k64, v64))  # unseen: whatever
    q64 = torch.where(see.any(3)[..., None], q64, 0.0)
    kr, vr = (t.repeat_interleave(G, 1) for t in (k64, v64))
    s = (q64 @ kr.transpose(2, 3).contiguous()) * scale
    s = s.masked_fill(~see, -math.inf)
    some = see.any(3, keepdim=True)
    p = torch.where(some, torch.softmax(s.masked_fill(~some, 0.0), -1), 0.0)
    o, oa = p @ vr, p @ vr.abs()
    slack = 2.0 ** -16
    # an error e of the scores (32-bit sums) is one of e of P
    se = (q64.abs() @ kr.abs().transpose(2, 3).contiguous()) * scale * 2.0 ** -20
    fuzz = slack + (se * p).amax(-1, keepdim=True) * 2
    res = {"out": (o, u * o.abs() + (u + fuzz) * oa + tiny * (1 + vr.abs().sum(2, keepdim=True)))}
    if grad is None:
        return res
    g = torch.where(some, grad.detach().double(), 0.0)
    ga = g.abs()
    dp = g @ vr.transpose(2, 3).contiguous()
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    mag = p * (ga @ vr.abs().transpose(2, 3).contiguous() + (ga * oa).sum(-1, keepdim=True))
    ds_err = u * ds.abs() + (slack + fuzz) * mag + p * u * (ga * oa).sum(-1, keepdim=True)
    far = 2.0 ** -38 * 2 * D * ga.amax() * vr.abs().amax() if tiny else 0.0

    def back(x):  # sums over the heads that share a key
        return x.reshape(B, Hk, G, Tk, D).sum(2)

    dq = scale * (ds @ kr)
    res["dq"] = (dq, u * dq.abs() + scale * ((ds_err + far * see) @ kr.abs()) + tiny)
    dk = scale * back(ds.transpose(2, 3).contiguous() @ q64)
    res["dk"] = (dk, u * dk.abs() + scale * back((ds_err + far * see).transpose(2, 3).contiguous() @ q64.abs()) + tiny)
    dv = back(p.transpose(2, 3).contiguous() @ g)
    pt = (u * p + fuzz * p + (2.0 ** -38 if tiny else 0.0) * see).transpose(2, 3).contiguous()
    res["dv"] = (dv, u * dv.abs() + back(pt @ ga) + tiny)
    return res


def check(got, want, names):
    for name, x in zip(names, got):
        value, bound = want[name]
        assert x.shape == value.shape, name
        off = (x.double() - value).abs()
        assert torch.isfinite(x).all(), name
        worst = (off / (bound + 1e-300)).max().item() if off.numel() else 0.0
        assert (off <= bound).all(), f"{name}: {worst:.2f} of the bound"
