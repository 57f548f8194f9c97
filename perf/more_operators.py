"""The operators with gradients, as cases that can be timed and compared: `run` makes the framework's calls where
`own` is true, and computes the same in elementary torch operations where it is false.

  attention  ress_amd.block_attention: softmax attention with a backward pass that forms the probabilities anew; dense,
             causal, over lengths, or over a map of 128-query x 64-key blocks as the block-sparse layers select it
  norm       ress_amd.layer_norm and ress_amd.add_layer_norm: layer norm with its backward pass, the latter of
             x + gamma * branch (a block's residual sum with LayerScale), which it returns beside the norm
  rotary     ress_amd.rotate: rotary positions of queries and keys by a RotaryTable (halves or interleaved pairs, the
             whole head or its first dims, one or two axes, tables scaled for long contexts), and their backward pass

A training case returns the gradients beside the outputs, as a training step's backward pass makes them.

Shapes: 518-pixel frames (37 x 37 patches and 5 special tokens: 1374 tokens a frame), 16 heads of 64 and a width of 1024;
and generic ones: grouped heads of 128, causal sequences of different lengths, single tokens.
"""

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
KS_Q, KS_K = 128, 64   # queries and keys of a block of the map
GRID = 37              # patches a side
SPECIAL = 5            # special tokens in front of a frame's patches
EPS = 1e-5


def _case(name, op, **kw):
    base = {"op": op, "dtype": "bfloat16", "grad": True}
    if op == "attention":
        # kept: the share of the map's blocks that a query block keeps (0: no map); empty: the map leaves some rows nothing;
        # packed: q, k and v are views of one projection's output
        base.update(batch=1, q_heads=16, kv_heads=16, dim=64, tq=1374, tk=1374, causal=False, ragged=False, kept=0.0,
                    empty=False, packed=False)
    elif op == "norm":
        # heads: rows are the heads of a projection's output, read in place; wide: weights in 32 bits
        base.update(rows=1374, width=1024, heads=0, branch=False, gamma=False, wide=False)
    else:
        base.update(batch=1, tokens=1374, q_heads=16, kv_heads=16, dim=64, axes=2, turned=64, layout="half",
                    scaling="none", packed=False)
    base.update(kw)
    if name:
        base["name"] = name
    return base


def listed():
    return [
        # one small image (11 x 11 patches and 5 special tokens) in a training step: the smallest, where latency counts
        _case("attention_small", "attention", tq=126, tk=126),
        # four frames' own attention in a training step, read from the projection's output
        _case("attention_frames", "attention", batch=4, packed=True),
        # the special tokens of 16 frames, which see every token: few rows, many keys
        _case("attention_special", "attention", tq=80, tk=21984),
        # a decoder's training step: causal, grouped heads of 128, a padded batch of different lengths
        _case("attention_causal", "attention", batch=4, q_heads=32, kv_heads=8, dim=128, tq=2048, tk=2048, causal=True,
              ragged=True, dtype="float16"),
        # a block-sparse global layer over 16 frames with 30% of the blocks kept, as a fine-tuning or calibration step has it
        _case("attention_sparse_16f", "attention", tq=16 * 1369, tk=21984, kept=0.3),
        # a single token's norm behind a residual sum: the smallest call
        _case("norm_token", "norm", rows=1, branch=True, gamma=True, grad=False),
        # one frame through a block's residual sum and norm in a training step
        _case("norm_frame", "norm", branch=True, gamma=True),
        # sixteen frames
        _case("norm_frames", "norm", rows=21984, branch=True, gamma=True),
        # the norm of four frames' queries, head by head, in a training step
        _case("norm_heads", "norm", rows=4 * 1374, width=64, heads=16),
        # one decoding step of a serving batch: interleaved pairs, a table scaled to 32 times the trained length
        _case("rotary_token", "rotary", batch=32, tokens=1, q_heads=32, kv_heads=8, dim=128, axes=1, turned=128,
              layout="interleaved", scaling="yarn", grad=False),
        # the patch grid's positions of 16 frames in a training step
        _case("rotary_frames", "rotary", tokens=21984, packed=True),
        # a decoder's training step, half of each head turned
        _case("rotary_part", "rotary", batch=4, tokens=4096, q_heads=32, kv_heads=8, dim=128, axes=1, turned=64,
              layout="interleaved", dtype="float16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """Another case of the same ranges; never more work than the block-sparse layer."""
    op = rng.choices(("attention", "norm", "rotary"), (50, 28, 22))[0]
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    if op == "norm":
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
        c = _case(None, op, rows=_log_int(rng, 1, 22000), width=rng.choice((64, 1024, _log_int(rng, 8, 8192))), dtype=dtype,
                  wide=rng.random() < 0.4, grad=rng.random() < 0.75)
        if c["width"] in (64, 128):
            c["heads"] = rng.choice((1, 8, 16))
        else:
            c["branch"] = rng.random() < 0.6
            c["gamma"] = c["branch"] and rng.random() < 0.6
        while c["rows"] * c["width"] * max(1, c["heads"]) > 30_000_000:
            c["rows"] //= 2
        return c
    dim = rng.choice((64, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 8)) if dim == 128 else rng.choice((2, 8, 16, 16, 24))
    heads = dict(kv_heads=kv_heads, q_heads=kv_heads * (rng.choice((1, 2, 4, 8)) if dim == 128 else rng.choice((1, 1, 1, 2))))
    batch = rng.choice((1, 1, 2, 4, 7))
    if op == "rotary":
        axes = 2 if dim == 64 and rng.random() < 0.6 else 1
        c = _case(None, op, batch=batch, tokens=_log_int(rng, 1, 22000), dim=dim, axes=axes, dtype=dtype,
                  turned=rng.choice((dim, dim, dim // 2, 24 * axes)), layout=rng.choice(("half", "interleaved")),
                  scaling=rng.choice(("none", "linear", "ntk", "yarn")) if axes == 1 else "none",
                  packed=rng.random() < 0.5 and heads["q_heads"] == kv_heads, grad=rng.random() < 0.7, **heads)
        while c["batch"] * c["tokens"] * (c["q_heads"] + c["kv_heads"]) * c["dim"] > 100_000_000:
            c["tokens"] = max(1, c["tokens"] // 2)
        return c
    tq, tk = _log_int(rng, 1, 22000), _log_int(rng, 4, 22000)
    kind = rng.choice(("dense", "same", "causal", "causal", "map", "map"))
    if kind in ("same", "causal"):
        tq = tk if rng.random() < 0.8 else max(1, tk // 3)
    c = _case(None, op, batch=batch, dim=dim, tq=tq, tk=tk, causal=kind == "causal",
              ragged=batch > 1 and rng.random() < 0.6, dtype=dtype,
              packed=tq == tk and rng.random() < 0.4 and heads["q_heads"] == kv_heads, grad=rng.random() < 0.8, **heads)
    if kind == "map":
        c.update(kept=rng.choice((0.1, 0.3, 0.6)), empty=rng.random() < 0.3)
    most = work(listed()[4])["flops"]
    while c["batch"] * c["q_heads"] * c["tq"] * c["tk"] > 3e9 or work(c)["flops"] > 0.7 * most:
        if c["batch"] > 2:
            c["batch"] //= 2
        elif c["tq"] == c["tk"]:
            c["tq"] = c["tk"] = max(1, c["tk"] // 2)
        elif c["tq"] > c["tk"]:
            c["tq"] //= 2
        else:
            c["tk"] //= 2
    return c


# ---- sizes ------------------------------------------------------------------
def _lengths(case):
    """(q_lens, k_lens) of each sequence, from the case alone."""
    B, tq, tk = case["batch"], case["tq"], case["tk"]
    if not case["ragged"]:
        return [tq] * B, [tk] * B
    share = [1.0 if b == 0 else ((b * 7919 + 61) % 97) / 97.0 for b in range(B)]
    ks = [int(round(tk * s)) for s in share]
    return ([k for k in ks] if tq == tk else [int(round(tq * s)) for s in share]), ks


def _kept(case):
    """Blocks of the map that a query block keeps, and the map's width."""
    nk = -(-case["tk"] // KS_K)
    return max(1, int(round(case["kept"] * nk))), nk


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["width"] * max(1, case["heads"])
        passes = (4 if case["branch"] else 2) + ((4 if case["branch"] else 2) if case["grad"] else 0)
        return {"bytes": size * n * passes, "flops": n * (8 + (14 if case["grad"] else 0))}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"] * (hq + hk) * d * (2 if case["grad"] else 1)
        return {"bytes": 2 * size * n, "flops": 3 * n * case["turned"] // d}
    pairs = 0
    for m, length in zip(*_lengths(case)):
        if case["causal"]:
            low = max(0, m - length)  # rows that see nothing
            pairs += (m - low) * length - (m - low) * (m - low - 1) // 2
        else:
            pairs += m * length
    rows, keys = (sum(x) for x in _lengths(case))
    if case["kept"]:
        n, nk = _kept(case)
        pairs = pairs * n // nk
    times = 2 if case["grad"] else 1  # the outputs' gradients beside q and o, those of k and v beside them
    return {"bytes": size * d * times * (2 * hq * rows + 2 * hk * keys), "flops": (14 if case["grad"] else 4) * hq * d * pairs}


# ---- inputs -----------------------------------------------------------------
def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _leaf(t, case):
    return t.detach().requires_grad_(case["grad"])


def _heads(case, tq, tk, g):
    """q, k, v (B, heads, tokens, dim): normalised keys with channels of unequal size and an offset shared by a head,
    queries that look for them, values of a smooth field; views of one buffer where the case is packed."""
    B, H, D, dt = case["batch"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    group = case["q_heads"] // H
    gain = torch.rand(H, 1, D, generator=g, device=DEV) + 0.5
    off = _rand(g, H, 1, D) * 0.5
    q = _rand(g, B, H * group, tq, D) * 1.5 / gain.repeat_interleave(group, 0)
    k, v = (_rand(g, B, H, tk, D) * gain + off for _ in range(2))
    if not case["packed"]:
        return [x.to(dt) for x in (q, k, v)]
    both = torch.stack([q, k, v], 2).to(dt)                       # (B, H, 3, T, D)
    both = both.permute(0, 3, 2, 1, 4).contiguous()               # (B, T, 3, H, D), as a projection writes it
    return list(both.permute(2, 0, 3, 1, 4).unbind(0))


def _map(case, g):
    """(B, heads, query blocks, key blocks): the best blocks of smooth scores that favour the near ones, as a layer selects
    them, in equal number for each row."""
    n, nk = _kept(case)
    nq = -(-case["tq"] // KS_Q)
    s = _rand(g, case["batch"], case["q_heads"], nq, nk)
    i = torch.arange(nq, device=DEV)[:, None] / nq - torch.arange(nk, device=DEV)[None] / nk
    s = s - 4.0 * i.abs()
    keep = torch.zeros_like(s, dtype=torch.bool).scatter_(3, s.topk(n, -1).indices, True)
    if case["empty"]:
        keep &= (torch.rand(case["batch"], case["q_heads"], nq, 1, generator=g, device=DEV) > 0.2)
    return keep


def _positions(case, g):
    B, n = case["batch"], case["tokens"]
    if case["axes"] == 1:
        most = _table_length(case)
        start = torch.randint(0, max(1, most - n + 1), (B, 1), generator=g, device=DEV)
        return start + torch.arange(n, device=DEV)[None]
    i = torch.arange(n, device=DEV) % (GRID * GRID + SPECIAL) - SPECIAL
    pos = torch.stack([torch.where(i < 0, 0, i // GRID + 1), torch.where(i < 0, 0, i % GRID + 1)], -1)
    return pos[None].expand(B, n, 2)


TRAINED = 4096  # positions that a scaled table's model was trained on
FACTORS = {"none": 1.0, "linear": 4.0, "ntk": 8.0, "yarn": 32.0}


def _table_length(case):
    return 64 if case["axes"] == 2 else max(32768, int(TRAINED * FACTORS[case["scaling"]]))


def _frequencies(case):
    """(angles a position of an axis' pairs, the factor on cosines and sines), in 64 bits."""
    d = case["turned"] // case["axes"]
    base = 10000.0 if case["axes"] == 1 else 100.0
    factor, kind = FACTORS[case["scaling"]], case["scaling"]
    if kind == "ntk":
        base *= factor ** (d / (d - 2))
    f = base ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    if kind == "linear":
        f = f / factor
    if kind != "yarn":
        return f, 1.0
    turns = TRAINED * f / (2 * math.pi)  # of a pair over the trained length: whole above 32, stretched below 1
    g = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return f * g + f / factor * (1.0 - g), 0.1 * math.log(factor) + 1.0


def _rope(case):
    from ress_amd import RotaryTable
    how = {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0},
           "yarn": {"type": "yarn", "factor": 32.0, "original": TRAINED}}[case["scaling"]]
    return RotaryTable(case["dim"], _table_length(case), base=10000.0 if case["axes"] == 1 else 100.0, axes=case["axes"],
                       device=DEV, layout=case["layout"], rotary_dim=case["turned"], scaling=how)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "norm":
        M, C, H = case["rows"], case["width"], case["heads"]
        wt = torch.float32 if case["wide"] else dt
        spread = 0.25 + 2.0 * torch.rand(C, generator=g, device=DEV)
        if H:  # the queries of a projection's output: (1, heads, rows, width), read in place
            x = (_rand(g, 1, M, 3, H, C) * spread + 0.3).to(dt).permute(2, 0, 3, 1, 4)[0]
        else:
            x = (_rand(g, M, C) * spread + 0.3 * _rand(g, C)).to(dt)
        s["x"] = _leaf(x, case)
        s["w"] = _leaf((1.0 + 0.2 * _rand(g, C)).to(wt), case)
        s["b"] = _leaf((0.1 * _rand(g, C)).to(wt), case)
        if case["branch"]:
            s["branch"] = _leaf((0.5 * _rand(g, M, C)).to(dt), case)
            if case["gamma"]:
                s["gamma"] = _leaf((0.3 * _rand(g, C) + 0.5).to(wt), case)
        if case["grad"]:
            s["dn"] = (0.02 * _rand(g, *x.shape)).to(dt)
            if case["branch"]:
                s["dh"] = (0.02 * _rand(g, *x.shape)).to(dt)
        return s
    if case["op"] == "rotary":
        q, k, _ = _heads(case, case["tokens"], case["tokens"], g)
        s["x"] = [_leaf(t, case) for t in (q, k)]
        s["pos"] = _positions(case, g)
        if case["grad"]:
            s["dy"] = [(0.02 * _rand(g, *t.shape)).to(dt) for t in (q, k)]
        if own:
            s["rope"] = _rope(case)
        else:
            f, gain = _frequencies(case)
            ang = torch.arange(_table_length(case), dtype=torch.float64, device=DEV)[:, None] * f
            s["rotary"] = torch.stack([ang.cos() * gain, ang.sin() * gain], 1).float()
        return s
    q, k, v = _heads(case, case["tq"], case["tk"], g)
    s["q"], s["k"], s["v"] = (_leaf(t, case) for t in (q, k, v))
    if case["grad"]:
        s["do"] = (0.02 * _rand(g, *q.shape)).to(dt)
    s["map"] = _map(case, g) if case["kept"] else None
    s["q_lens"] = s["k_lens"] = None
    if case["ragged"]:
        s["q_lens"], s["k_lens"] = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in _lengths(case))
    return s


# ---- the operators ----------------------------------------------------------
def _attention_plain(s):
    case = s["case"]
    B, Hq, Hk, D, tq, tk = (case[n] for n in ("batch", "q_heads", "kv_heads", "dim", "tq", "tk"))
    dt, group, scale = DTYPES[case["dtype"]], case["q_heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    q, k, v = (s[n].detach() for n in "qkv")
    out = torch.empty(B, Hq, tq, D, dtype=dt, device=DEV)
    if case["grad"]:
        dq = torch.empty(B, Hq, tq, D, dtype=dt, device=DEV)
        dk, dv = (torch.empty(B, Hk, tk, D, dtype=dt, device=DEV) for _ in range(2))
    rows, keys = torch.arange(tq, device=DEV), torch.arange(tk, device=DEV)
    step = max(1, min(Hk, int(5e8 / (group * tq * tk))))  # key/value heads at a time, to bound the memory
    for b in range(B):
        seen = torch.ones(tq, tk, dtype=torch.bool, device=DEV)
        shift = tk - tq
        if case["ragged"]:
            m, length = s["q_lens"][b], s["k_lens"][b]
            shift = length - m
            seen = (rows < m)[:, None] & (keys < length)[None]
        if case["causal"]:
            seen = seen & (keys[None] <= rows[:, None] + shift)
        for h in range(0, Hk, step):
            n = min(step, Hk - h)
            kh, vh = k[b, h:h + n].float()[:, None], v[b, h:h + n].float()[:, None]
            hs = slice(h * group, (h + n) * group)
            qh = q[b, hs].float().reshape(n, group, tq, D)
            see = seen[None, None]
            if s["map"] is not None:
                keep = s["map"][b, hs].repeat_interleave(KS_Q, 1)[:, :tq].repeat_interleave(KS_K, 2)[:, :, :tk]
                see = see & keep.reshape(n, group, tq, tk)
                del keep
            kt = kh.transpose(2, 3).contiguous()
            p = torch.matmul(qh * scale, kt)
            p.masked_fill_(~see, -math.inf)
            p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
            total = p.sum(-1, keepdim=True)
            p.mul_(torch.where(total > 0, 1.0 / total, 0.0))
            o = torch.matmul(p, vh)
            out[b, hs] = o.reshape(n * group, tq, D).to(dt)
            if not case["grad"]:
                continue
            do = s["do"][b, hs].float().reshape(n, group, tq, D)
            ds = torch.matmul(do, vh.transpose(2, 3).contiguous())
            ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            dv[b, h:h + n] = torch.matmul(p.transpose(2, 3).contiguous(), do).sum(1).to(dt)
            del p
            dq[b, hs] = torch.matmul(ds, kh).reshape(n * group, tq, D).to(dt)
            dk[b, h:h + n] = torch.matmul(ds.transpose(2, 3).contiguous(), qh).sum(1).to(dt)
            del ds
    return [out, dq, dk, dv] if case["grad"] else [out]


def _norm_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, w, b = (s[n].detach().float() for n in ("x", "w", "b"))
    outs = []
    if case["branch"]:
        branch = s["branch"].detach().float()
        gamma = s["gamma"].detach().float() if case["gamma"] else None
        h = (x + branch * gamma if case["gamma"] else x + branch).to(dt)  # the norm is that of the sum as it is returned
        outs.append(h)
        x = h.float()
    c = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    xhat = c * rstd
    outs.append((xhat * w + b).to(dt))
    if not case["grad"]:
        return outs
    dn = s["dn"].float()
    g = dn * w
    dx = (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True)) * rstd
    lead = tuple(range(x.dim() - 1))
    ends = [(dn * xhat).sum(lead).to(s["w"].dtype), dn.sum(lead).to(s["b"].dtype)]
    if not case["branch"]:
        return outs + [dx.to(dt)] + ends
    dx = dx + s["dh"].float()
    if not case["gamma"]:
        return outs + [dx.to(dt), dx.to(dt)] + ends
    return outs + [dx.to(dt), (dx * gamma).to(dt), (dx * branch).sum(lead).to(s["gamma"].dtype)] + ends


def _turned(x, pos, rotary, case, sign):
    d, n = case["turned"] // case["axes"], case["turned"]
    parts = []
    y = x.float()
    for a, part in enumerate(y[..., :n].split(d, -1)):
        cs = rotary[pos if case["axes"] == 1 else pos[..., a]][:, None]  # (B, 1, tokens, 2, d/2)
        c, si = cs[..., 0, :], cs[..., 1, :] * sign
        if case["layout"] == "half":
            x1, x2 = part[..., : d // 2], part[..., d // 2:]
            parts += [x1 * c - x2 * si, x2 * c + x1 * si]
        else:
            x1, x2 = part[..., 0::2], part[..., 1::2]
            parts.append(torch.stack([x1 * c - x2 * si, x2 * c + x1 * si], -1).flatten(-2))
    return torch.cat(parts + [y[..., n:]], -1).to(x.dtype)


def _rotary_plain(s):
    case = s["case"]
    outs = [_turned(x.detach(), s["pos"], s["rotary"], case, 1.0) for x in s["x"]]
    if case["grad"]:  # turned back: the transpose of a rotation
        outs += [_turned(dy, s["pos"], s["rotary"], case, -1.0) for dy in s["dy"]]
    return outs


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"attention": _attention_plain, "norm": _norm_plain, "rotary": _rotary_plain}[case["op"]](s)
    import ress_amd as ress
    if case["op"] == "attention":
        out = ress.block_attention(s["q"], s["k"], s["v"], block_map=s["map"], causal=case["causal"], q_lens=s["q_lens"],
                                   k_lens=s["k_lens"])
        if not case["grad"]:
            return [out]
        return [out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])]
    if case["op"] == "rotary":
        outs = ress.rotate(s["x"], s["pos"], s["rope"])
        return [*outs, *torch.autograd.grad(outs, s["x"], s["dy"])] if case["grad"] else list(outs)
    if not case["branch"]:
        n = ress.layer_norm(s["x"], s["w"], s["b"], eps=EPS)
        return [n, *torch.autograd.grad(n, (s["x"], s["w"], s["b"]), s["dn"])] if case["grad"] else [n]
    outs = ress.add_layer_norm(s["x"], s["branch"], s.get("gamma"), s["w"], s["b"], eps=EPS)
    if not case["grad"]:
        return list(outs)
    leaves = [s[n] for n in ("x", "branch", "gamma", "w", "b") if n in s]
    return [*outs, *torch.autograd.grad(outs, leaves, (s["dh"], s["dn"]))]


# ---- the same in 64 bits, gradients by differentiating the definition -------
def _attention_exact(s, case):
    B, Hq, Hk, D, tq, tk = (case[n] for n in ("batch", "q_heads", "kv_heads", "dim", "tq", "tk"))
    group = Hq // Hk
    f64 = dict(dtype=torch.float64, device=DEV)
    out, dq = torch.zeros(B, Hq, tq, D, **f64), torch.zeros(B, Hq, tq, D, **f64)
    dk, dv = torch.zeros(B, Hk, tk, D, **f64), torch.zeros(B, Hk, tk, D, **f64)
    for b, (m, length) in enumerate(zip(*_lengths(case))):
        if m == 0 or length == 0:
            continue
        for h in range(Hq):
            q, k, v = (s[n].detach()[b, i, :e].double().requires_grad_(case["grad"])
                       for n, i, e in (("q", h, m), ("k", h // group, length), ("v", h // group, length)))
            hide = None
            if case["causal"]:
                hide = torch.ones(m, length, dtype=torch.bool, device=DEV).triu(length - m + 1)
            if s["map"] is not None:
                keep = s["map"][b, h][torch.arange(m, device=DEV) // KS_Q][:, torch.arange(length, device=DEV) // KS_K]
                hide = ~keep if hide is None else hide | ~keep
            with torch.set_grad_enabled(case["grad"]):
                a = q @ k.T / math.sqrt(D)
                if hide is not None:
                    a = a.masked_fill(hide, -math.inf)
                    a = a.masked_fill(hide.all(1, keepdim=True), 0.0)
                o = torch.softmax(a, -1) @ v
                if hide is not None:
                    o = o.masked_fill(hide.all(1, keepdim=True), 0.0)
            out[b, h, :m] = o.detach()
            if case["grad"]:
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["do"][b, h, :m].double())
                dq[b, h, :m] = gq
                dk[b, h // group, :length] += gk
                dv[b, h // group, :length] += gv
            del a, o
    return [out, dq, dk, dv] if case["grad"] else [out]


def _norm_exact(s, case):
    x, w, b = (s[n].detach().double().requires_grad_(case["grad"]) for n in ("x", "w", "b"))
    outs, h = [], x
    if case["branch"]:
        branch = s["branch"].detach().double()
        gamma = s["gamma"].detach().double() if case["gamma"] else torch.ones((), dtype=torch.float64, device=DEV)
        outs.append(x.detach() + gamma * branch)
        h = outs[0].to(DTYPES[case["dtype"]]).double().requires_grad_(case["grad"])
    with torch.set_grad_enabled(case["grad"]):
        var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
        n = (h - mean) / (var + EPS).sqrt() * w + b
    outs.append(n.detach())
    if not case["grad"]:
        return outs
    gh, gw, gb = torch.autograd.grad(n, (h, w, b), s["dn"].double())
    if not case["branch"]:
        return outs + [gh, gw, gb]
    gh = gh + s["dh"].double()
    ends = [gh, gh * gamma] + ([(gh * branch).sum(0)] if case["gamma"] else [])
    return outs + ends + [gw, gb]


def _rotary_exact(s, case):
    f, gain = _frequencies(case)
    d, n = case["turned"] // case["axes"], case["turned"]
    outs = []
    for turn, xs in ((1.0, s["x"]), (-1.0, s.get("dy", ()))):
        for x in xs:
            x, parts = x.detach().double(), []
            for a in range(case["axes"]):
                p = (s["pos"] if case["axes"] == 1 else s["pos"][..., a]).double()[:, None, :, None]
                y = x[..., a * d:(a + 1) * d]
                y = y.unflatten(-1, (2, d // 2)) if case["layout"] == "half" else y.unflatten(-1, (d // 2, 2)).transpose(-1, -2)
                z = torch.complex(y[..., 0, :], y[..., 1, :]) * torch.polar(torch.full_like(p * f, gain), turn * p * f)
                y = torch.stack([z.real, z.imag], -2)
                parts.append((y if case["layout"] == "half" else y.transpose(-1, -2)).flatten(-2))
            outs.append(torch.cat(parts + [x[..., n:]], -1))
    return outs


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _attention_exact, "norm": _norm_exact, "rotary": _rotary_exact}[case["op"]](s, case)
