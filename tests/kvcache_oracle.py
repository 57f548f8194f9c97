"""What a PagedKVCache holds and what attention over it is, in 64 bits, from its buffers."""

import math

import torch

PAGE = 64


def v_token(p):
    """The token of place p of a value row (csrc/kvcache.h)."""
    return ((p >> 3) & 1) * 32 + ((p >> 2) & 1) * 16 + (p >> 4) * 4 + (p & 3)


V_ORDER = torch.tensor(sorted(range(PAGE), key=v_token))  # place of token 0, 1, ...


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def held(cache, slot):
    """(k, v) (H, length, D) float64 of one slot on the CPU, straight from codes, scales and tails."""
    L = int(cache.lens[slot])
    full, left = L // PAGE, L % PAGE
    ids = cache.table[slot, :full].long().cpu()
    k = cache.k_codes.cpu().double()[ids] * cache.k_scale.cpu().double()[ids][..., None, None]      # (P, H, 64, D)
    v = cache.v_codes.cpu().double()[ids] * cache.v_scale.cpu().double()[ids][..., None, None]      # (P, H, D, 64)
    v = v[..., V_ORDER].transpose(-1, -2)
    H, D = cache.kv_heads, cache.head_dim
    k = k.transpose(0, 1).reshape(H, full * PAGE, D)
    v = v.transpose(0, 1).reshape(H, full * PAGE, D)
    tk = cache.tail_k[slot].cpu().double()[:, :left]
    tv = cache.tail_v[slot].cpu().double()[..., V_ORDER].transpose(-1, -2)[:, :left]
    return torch.cat([k, tk], 1), torch.cat([v, tv], 1)


def attention(q, k, v, n_new, causal, scale=None):
    """(out, bound_v, spread): softmax(scale q K^T) V of q (Hq, n, D) over k, v (H, L, D) in 64 bits for the
    first n_new rows; bound_v = sum_j p_j |v_j| and spread = sum_d |q_d| max_j |k_jd| * scale, what rounding
    errors of P and of the scores are measured in."""
    Hq, n, D = q.shape
    H, L, _ = k.shape
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    q = q.double().cpu()
    out, size = torch.zeros(Hq, n, D, dtype=torch.float64), torch.zeros(Hq, n, D, dtype=torch.float64)
    spread = torch.zeros(Hq, n, 1, dtype=torch.float64)
    for h in range(Hq):
        a = q[h] @ k[h // G].T * scale
        if causal:
            seen = torch.arange(L)[None] <= (L - n_new + torch.arange(n))[:, None]
            a = a.masked_fill(~seen, -math.inf)
        a[n_new:] = -math.inf
        if L:
            m = a.amax(-1, keepdim=True)
            p = torch.exp(a - m.clamp(min=-1e300))
            p[~(m > -math.inf).expand_as(p) & ~m.isnan().expand_as(p)] = 0
            s = p.sum(-1, keepdim=True)
            vv = v[h // G]
            out[h] = torch.where(s == 0, 0, (p @ vv) / s)
            size[h] = torch.where(s == 0, 0, (p @ vv.abs()) / s)
            spread[h, :, 0] = (q[h].abs() * k[h // G].abs().amax(0)).sum(-1) * scale
    return out, size, spread


def tolerance(out, size, spread, dtype, L):
    """|error| allowed: P is rounded to 16 bits (half a step each, in the product with V: times sum p |v|, and in the
    sum that it is divided by: times |out|), in fp16 the values too (a step of the type's subnormals apart at most:
    `tiny`), and the output once more; the scores, their exponential (2 units of 2^-23) and the sums are fp32: a score of D = 128
    products and two multiplications is off by at most 130 * 2^-24 * spread, which its exponential turns into
    that relative error, and a sum of L terms by L * 2^-24 (numerator and denominator)."""
    u = half_step(dtype)
    rel = (2 if dtype == torch.float16 else 1) * u + 2 * (130 * 2.0 ** -24 * spread + 2.0 ** -22) + 2 * (L + 64) * 2.0 ** -24
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a subnormal step of the output
    return rel * size + 2 * u * out.abs() + tiny
