"""Operators with a backward pass: what a block of the model runs in a training or calibration step.

    out = block_attention(q, k, v, block_map=kept)            # softmax attention over a map of 128-query x 64-key blocks
    h, n = add_layer_norm(x, branch, gamma, weight, bias)     # x + gamma * branch, and its layer norm
    q, k = rotate((q, k), pos, rope)                          # rotary positions by a RotaryTable

The block-sparse layers run without gradients. Calibration tables (a head's Fisher scores) and fine-tuning under a fixed
map need them; ress_amd.training puts these operators into a model's blocks.

Every operator works on torch's current stream of its operands' device, waits for nothing and repeats bit for bit: no sum
is made by atomics. Gradients are formed once (no second derivatives), in the operands' types with 32-bit sums.
Operands with strides that a kernel cannot take are copied first. The reference has no counterpart: its kernels have no
backward pass.

In a captured graph: torch accumulates a leaf's gradient on the stream on which the leaf entered the oldest graph that still
lives. Where that is an eager one of the default stream, capturing the backward pass would end the process: a call with such
a leaf is refused inside a capture (delete the eager result first, or run it on a side stream).
"""

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from ress_amd import _lib

DTYPES = {torch.bfloat16: 1, torch.float16: 2}
Q_BLOCK, K_BLOCK = 128, 64
MOST_TOKENS, MOST_MAPPED = 1 << 26, 1 << 20
MOST_STRIDE = 1 << 24


class _Strided(ctypes.Structure):
    """ress_strided of include/ress_hip.h."""

    _fields_ = [("data", ctypes.c_void_p), ("sb", ctypes.c_longlong), ("sh", ctypes.c_longlong), ("st", ctypes.c_longlong)]


class _Rows(ctypes.Structure):
    """ress_rows."""

    _fields_ = [("data", ctypes.c_void_p), ("s0", ctypes.c_longlong), ("s1", ctypes.c_longlong), ("s2", ctypes.c_longlong)]


class _NormArgs(ctypes.Structure):
    """ress_layer_norm."""

    _fields_ = ([("x", _Rows), ("branch", _Rows)] + [(n, ctypes.c_int) for n in ("n0", "n1", "n2", "C", "dtype", "wide")]
                + [(n, ctypes.c_void_p) for n in ("gamma", "weight", "bias", "sum", "out", "mean", "rstd")] + [("eps", ctypes.c_float)])


class _RotaryArgs(ctypes.Structure):
    """ress_rotary."""

    _fields_ = ([("x", _Strided * 2), ("y", _Strided * 2), ("heads", ctypes.c_int * 2)]
                + [(n, ctypes.c_int) for n in ("B", "n", "head_dim", "dtype", "axes", "rotary_dim", "interleaved", "inverse")]
                + [("pos", ctypes.c_void_p), ("pos_sb", ctypes.c_longlong), ("pos_st", ctypes.c_longlong),
                   ("pos_sa", ctypes.c_longlong), ("table", ctypes.c_void_p), ("positions", ctypes.c_int), ("status", ctypes.c_void_p)])


class _AttnArgs(ctypes.Structure):
    """ress_block_attn of include/ress_hip.h."""

    _fields_ = ([(n, _Strided) for n in ("q", "k", "v", "out")]
                + [(n, ctypes.c_int) for n in ("B", "q_heads", "kv_heads", "Tq", "Tk", "head_dim", "dtype", "causal")]
                + [("q_lens", ctypes.c_void_p), ("k_lens", ctypes.c_void_p), ("map", ctypes.c_void_p)]
                + [(n, ctypes.c_longlong) for n in ("map_sb", "map_sh", "map_sq", "map_sk")]
                + [("lse", ctypes.c_void_p), ("rest", ctypes.c_void_p), ("scale", ctypes.c_float)])


def _strides(t):
    """Strides (batch, heads, tokens) that the kernels take of t (B, H, T, D), those of single entries in their place; None
    where they do not."""
    B, H, T, D = t.shape
    sb, sh, st, sd = t.stride()
    sb, sh, st = sb if B > 1 else 0, sh if H > 1 else 0, st if T > 1 else D
    if sd != 1 or st < D or st >= MOST_STRIDE or (sb | sh | st) & 7 or t.data_ptr() & 15:
        return None
    return sb, sh, st


def _ready(t):
    return t if t.numel() == 0 or _strides(t) is not None else t.clone(memory_format=torch.contiguous_format)


def _strided(t):
    return _Strided(t.data_ptr(), *(_strides(t) if t.numel() else (0, 0, t.shape[3])))


def _capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _differentiates(*tensors):
    """Whether a call on these tensors makes a graph; refuses leaves whose gradients cannot be captured."""
    if not torch.is_grad_enabled():
        return False
    leaves = [t for t in tensors if t is not None and t.requires_grad]
    if not leaves:
        return False
    capturing = _capturing()
    if not capturing and _lib.stream_handle(leaves[0].device):
        return True
    for t in leaves:
        if t.is_leaf:
            seen = torch.autograd.graph.get_gradient_edge(t).node.metadata  # lives as long as a graph with the leaf
            if not capturing:
                seen["ress_default_stream"] = True
            elif "ress_default_stream" in seen:
                raise RuntimeError("inside a graph capture: a result of the same leaves from outside of it, on the default "
                                   "stream, is still alive; delete it first")
    return True


def _lens(lens, name, B, T, device):
    if lens is None:
        return None
    if not torch.is_tensor(lens):
        lens = [int(x) for x in lens]
        if len(lens) != B or any(not 0 <= x <= T for x in lens):
            raise ValueError(f"{name} must be {B} counts of 0..{T}, got {lens}")
        if _capturing():
            raise RuntimeError(f"inside a graph capture {name} must be an int32 tensor made before it")
        return torch.tensor(lens, dtype=torch.int32, device=device)
    if lens.device != device or lens.dtype != torch.int32 or tuple(lens.shape) != (B,):
        raise ValueError(f"{name} must be ({B},) int32 on {device}, got {tuple(lens.shape)} {lens.dtype} on {lens.device}")
    return lens.contiguous()


def _arguments(q, k, v, out, block_map, causal, q_lens, k_lens, scale, lse, rest):
    B, Hq, Tq, D = q.shape
    P = _lib.ptr
    ms = block_map.stride() if block_map is not None else (0, 0, 0, 0)
    return _AttnArgs(_strided(q), _strided(k), _strided(v), _strided(out), B, Hq, k.shape[1], Tq, k.shape[2], D, DTYPES[q.dtype],
                     1 if causal else 0, P(q_lens), P(k_lens), P(block_map), *ms, P(lse), P(rest), scale)


def _attend(q, k, v, block_map, causal, q_lens, k_lens, scale, grads):
    out = torch.empty_like(q)
    if out.numel() and _strides(out) is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = rest = None
    if grads:
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
        rest = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.numel():
        args = _arguments(q, k, v, out, block_map, causal, q_lens, k_lens, scale, lse, rest)
        _lib.call_on(q.device, "ress_block_attn_fwd", ctypes.addressof(args))
    return out, lse, rest


class _BlockAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, block_map, causal, q_lens, k_lens, scale):
        q, k, v = _ready(q), _ready(k), _ready(v)
        out, lse, rest = _attend(q, k, v, block_map, causal, q_lens, k_lens, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, rest, block_map, q_lens, k_lens)
        ctx.how = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, rest, block_map, q_lens, k_lens = ctx.saved_tensors
        causal, scale = ctx.how
        grad = _ready(grad)
        grads = [torch.empty_like(t) for t in (q, k, v)]
        grads = [t if t.numel() == 0 or _strides(t) is not None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
                 for t in grads]
        args = _arguments(q, k, v, out, block_map, causal, q_lens, k_lens, scale, lse, rest)
        size = _lib.lib().ress_block_attn_bwd_workspace_size(ctypes.addressof(args))
        work = torch.empty(size, dtype=torch.uint8, device=q.device)
        g = [_strided(t) for t in (grad, *grads)]
        _lib.call_on(q.device, "ress_block_attn_bwd", ctypes.addressof(args), *(ctypes.addressof(t) for t in g), _lib.ptr(work),
                     size)
        return (*grads, None, None, None, None, None)


def _check_attention(q, k, v, block_map):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not torch.is_tensor(t) or not t.is_cuda:
            raise RuntimeError(f"{name} must be a device tensor (the attention runs only on the GPU)")
        if t.dtype not in DTYPES:
            raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must be {q.dtype} on {q.device} like q, got {t.dtype} on {t.device}")
        if t.dim() != 4:
            raise ValueError(f"{name} must be (B, heads, tokens, head_dim), got {tuple(t.shape)}")
    B, Hq, Tq, D = q.shape
    Hk, Tk = k.shape[1], k.shape[2]
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    if k.shape != (B, Hk, Tk, D) or v.shape != k.shape:
        raise ValueError(f"k and v must be ({B}, kv_heads, tokens, {D}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if Hk == 0 or Hq % Hk:
        raise ValueError(f"q must have a multiple of k's heads, got {Hq} and {Hk}")
    if max(Tq, Tk) > MOST_TOKENS:
        raise ValueError(f"at most {MOST_TOKENS} tokens, got {Tq} and {Tk}")
    if block_map is not None:
        want = (-(-Tq // Q_BLOCK), -(-Tk // K_BLOCK))
        if not torch.is_tensor(block_map) or block_map.dtype not in (torch.bool, torch.uint8) or block_map.device != q.device:
            raise ValueError(f"block_map must be a bool or uint8 tensor on {q.device}")
        if (block_map.dim() != 4 or tuple(block_map.shape[2:]) != want or block_map.shape[0] not in (1, B)
                or block_map.shape[1] not in (1, Hq)):
            raise ValueError(f"block_map must be ({B} or 1, {Hq} or 1, {want[0]}, {want[1]}): {Q_BLOCK}-query x {K_BLOCK}-key "
                             f"blocks, got {tuple(block_map.shape)}")
        if max(Tq, Tk) > MOST_MAPPED:
            raise ValueError(f"at most {MOST_MAPPED} tokens under a block_map, got {Tq} and {Tk}")


def block_attention(q, k, v, block_map=None, causal=False, q_lens=None, k_lens=None, scale=None):
    """softmax(scale q k^T) v, (B, heads, tokens, head_dim), with a backward pass to q, k and v. q (B, heads, Tq, head_dim), k and
    v (B, kv_heads, Tk, head_dim), bfloat16 or float16, head_dim 64 or 128, heads a multiple of kv_heads (query head h
    reads key/value head h / (heads / kv_heads)), any strides. scale: 1/sqrt(head_dim).

    A row sees the keys below its sequence's k_lens[b]; with causal=True of these the keys up to its own token, the rows being the
    last q_lens[b] of the sequence's k_lens[b] tokens; with a block_map (B or 1, heads or 1, ceil(Tq / 128), ceil(Tk / 64)),
    bool or uint8, of these the keys of blocks that it keeps (the final_map of a block-sparse layer is one). q_lens and
    k_lens: (B,) int32 on the device (clamped into the tensors), or lists. Rows that see nothing and rows from q_lens[b] on are zero,
    in the output and the gradients. Tokens past the lengths and blocks that are dropped reach nothing, whatever they
    hold; a key or value that is not finite makes NaN of the rows that see its block, in a causal block also of those that see
    only a part of it.

    The probabilities, formed anew in the backward pass, and the scores' gradients are rounded to the operands' type before
    they are multiplied; sums, maxima and the softmax's statistics are fp32. A forward pass for gradients keeps, beside its
    operands and output, a tensor of the output's size (what its rounding took) and 4 bytes a row."""
    _check_attention(q, k, v, block_map)
    B, Hq, Tq, D = q.shape
    Tk = k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    q_lens, k_lens = _lens(q_lens, "q_lens", B, Tq, q.device), _lens(k_lens, "k_lens", B, Tk, q.device)
    if block_map is not None:
        block_map = block_map.expand(B, Hq, -1, -1)
    if _differentiates(q, k, v):
        return _BlockAttention.apply(q, k, v, block_map, causal, q_lens, k_lens, scale)
    return _attend(_ready(q), _ready(k), _ready(v), block_map, causal, q_lens, k_lens, scale, False)[0]


# ---- layer norm ------------------------------------------------------------------
NORM_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST_WIDTH, MOST_ROWS = 8192, (1 << 31) - 1


def _rows_of(tensors):
    """(n0, n1, n2, {id: strides}) of rows (..., C) of several tensors of one shape; the tensors themselves, copied where
    their rows cannot be taken in place."""
    shape = tensors[0].shape
    lead = [i for i in range(len(shape) - 1) if shape[i] > 1]
    if all(t.is_contiguous() for t in tensors) or len(lead) > 3 or shape[-1] == 0:
        tensors = [t.contiguous() for t in tensors]
        rows = 1
        for n in shape[:-1]:
            rows *= n
        return (rows, 1, 1), tensors, [(shape[-1], 0, 0)] * len(tensors)
    tensors = [t if t.stride(-1) == 1 or shape[-1] == 1 else t.contiguous() for t in tensors]
    pad = 3 - len(lead)
    sizes = tuple([1] * pad + [shape[i] for i in lead])
    return sizes, tensors, [tuple([0] * pad + [t.stride(i) for i in lead]) for t in tensors]


def _norm_args(sizes, C, x, xs, branch, bs, gamma, weight, bias, total, out, mean, rstd, eps):
    P = _lib.ptr
    # the axis that varies fastest last; rows of one axis go first
    if sizes[0] == 1 and sizes[1] == 1:
        sizes, xs, bs = (sizes[2], 1, 1), (xs[2], 0, 0), (bs[2], 0, 0)
    wide = any(w is not None and w.dtype is torch.float32 for w in (gamma, weight, bias))
    return _NormArgs(_Rows(P(x), *xs), _Rows(P(branch), *bs), *sizes, C, NORM_DTYPES[x.dtype], 1 if wide else 0, P(gamma), P(weight),
                     P(bias), P(total), P(out), P(mean), P(rstd), eps)


def _normalise(x, branch, gamma, weight, bias, eps, grads):
    """(sum or None, n, mean, rstd)"""
    operands = [x] if branch is None else [x, branch]
    sizes, operands, strides = _rows_of(operands)
    C = x.shape[-1]
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if branch is not None else None
    mean = rstd = None
    if grads:
        mean, rstd = torch.empty((2, sizes[0] * sizes[1] * sizes[2]), dtype=torch.float32, device=x.device)
    if out.numel():
        args = _norm_args(sizes, C, operands[0], strides[0], operands[1] if branch is not None else None,
                          strides[-1], gamma, weight, bias, total, out, mean, rstd, eps)
        _lib.call_on(x.device, "ress_layer_norm_fwd", ctypes.addressof(args))
    return total, out, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gamma, weight, bias, eps):
        ctx.set_materialize_grads(False)
        total, out, mean, rstd = _normalise(x, branch, gamma, weight, bias, eps, True)
        ctx.save_for_backward(x if branch is None else total, branch, gamma, weight, bias, mean, rstd)
        ctx.eps = eps
        return out if branch is None else (total, out)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        h, branch, gamma, weight, bias, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dh, dn = grads if branch is not None else (None, grads[0])
        if dh is None and dn is None:
            return (None,) * 6

        def make(like, wanted):
            return torch.empty(like.shape, dtype=like.dtype, device=like.device) if wanted and like is not None else None

        dx = make(h, need[0] or (need[1] and gamma is None))
        dbranch = make(h, need[1] and gamma is not None)
        dgamma, dweight, dbias = make(gamma, need[2]), make(weight, need[3]), make(bias, need[4])
        ends = [t for t in (dgamma, dweight, dbias) if t is not None]
        if h.numel() == 0:
            for t in ends:
                t.zero_()
        else:
            given = [t for t in (h, branch, dh, dn) if t is not None]
            sizes, given, strides = _rows_of(given)
            at = dict(zip([n for n, t in (("h", h), ("branch", branch), ("dh", dh), ("dn", dn)) if t is not None],
                          zip(given, strides)))
            none = (None, (0, 0, 0))
            x_, xs = at["h"]
            b_, bs = at.get("branch", none)
            args = _norm_args(sizes, h.shape[-1], x_, xs, b_, bs, gamma, weight, bias, None, None, mean, rstd, ctx.eps)
            one = sizes[0] == 1 and sizes[1] == 1

            def rows(name):
                t, s = at.get(name, none)
                return ctypes.byref(_Rows(t.data_ptr(), *((s[2], 0, 0) if one else s))) if t is not None else None

            size = _lib.lib().ress_layer_norm_bwd_workspace_size(ctypes.addressof(args)) if ends else 0
            work = torch.empty(size, dtype=torch.uint8, device=h.device) if size else None
            P = _lib.ptr
            _lib.call_on(h.device, "ress_layer_norm_bwd", ctypes.addressof(args), rows("dn"), rows("dh"), P(dx), P(dbranch),
                         P(dgamma), P(dweight), P(dbias), P(work), size)
        if need[1] and gamma is None:
            dbranch = dx
        return dx if need[0] else None, dbranch, dgamma, dweight, dbias, None


def _check_norm(x, branch, gamma, weight, bias, eps):
    if not torch.is_tensor(x) or not x.is_cuda:
        raise RuntimeError("x must be a device tensor (the norm runs only on the GPU)")
    if x.dtype not in NORM_DTYPES:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MOST_WIDTH:
        raise ValueError(f"x must have a last dim of 1 to {MOST_WIDTH}, got {tuple(x.shape)}")
    if x.numel() > MOST_ROWS * x.shape[-1]:
        raise ValueError(f"x must have at most {MOST_ROWS} rows, got {tuple(x.shape)}")
    C = x.shape[-1]
    if branch is not None:
        if not torch.is_tensor(branch) or branch.device != x.device or branch.dtype != x.dtype or branch.shape != x.shape:
            raise ValueError(f"branch must be {tuple(x.shape)} {x.dtype} on {x.device} like x")
    given = [(n, t) for n, t in (("gamma", gamma), ("weight", weight), ("bias", bias)) if t is not None]
    for name, t in given:
        if not torch.is_tensor(t) or t.device != x.device or tuple(t.shape) != (C,) or t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be ({C},) {x.dtype} or float32 on {x.device}")
        if t.dtype != given[0][1].dtype:
            raise ValueError(f"{', '.join(n for n, _ in given)} must have one type")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must not be negative, got {eps}")


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dim (up to 8192), in x's type (bfloat16, float16 or float32), with a
    backward pass. x (..., C), any strides; weight and bias (C,) of x's type or, both, float32 (None: 1 and 0). Statistics,
    kept for the backward pass (8 bytes a row), and sums are fp32; the result is contiguous."""
    eps = float(eps)
    _check_norm(x, None, None, weight, bias, eps)
    weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
    if _differentiates(x, weight, bias):
        return _LayerNorm.apply(x, None, None, weight, bias, eps)
    return _normalise(x, None, None, weight, bias, eps, False)[1]


def add_layer_norm(x, branch, gamma=None, weight=None, bias=None, eps=1e-5):
    """(h, n): the residual sum h = x + gamma * branch and n = layer_norm(h, weight, bias, eps), in one pass over x and branch and with
    one backward pass, to all five. branch: shape and type of x; gamma (a LayerScale), weight, bias: (C,), of x's type or, all of
    them, float32 (None: 1, 1 and 0). The norm is that of h as it is returned, rounded to its type."""
    eps = float(eps)
    if branch is None:
        raise ValueError("branch is missing (layer_norm takes x alone)")
    _check_norm(x, branch, gamma, weight, bias, eps)
    gamma, weight, bias = (t if t is None else t.contiguous() for t in (gamma, weight, bias))
    if _differentiates(x, branch, gamma, weight, bias):
        return _LayerNorm.apply(x, branch, gamma, weight, bias, eps)
    return _normalise(x, branch, gamma, weight, bias, eps, False)[:2]


# ---- rotary positions ------------------------------------------------------------
def _turn(xs, pos, rope, inverse):
    """The operands turned (one or two), each in a tensor laid out like it."""
    ys = []
    for x in xs:
        y = torch.empty_like(x)
        ys.append(y if y.stride(3) == 1 or y.numel() == 0 else torch.empty(x.shape, dtype=x.dtype, device=x.device))
    B, _, n, D = xs[0].shape
    if n and B and any(x.shape[1] for x in xs):
        xs = [x if x.stride(3) == 1 else x.contiguous() for x in xs]

        def two(ts):
            return (_Strided * 2)(*(_Strided(t.data_ptr(), *t.stride()[:3]) for t in ts))

        args = _RotaryArgs(two(xs), two(ys), (ctypes.c_int * 2)(*(x.shape[1] for x in xs)), B, n, D, DTYPES[xs[0].dtype], rope.axes,
                           rope.rotary_dim, 1 if rope.layout == "interleaved" else 0, 1 if inverse else 0, pos.data_ptr(),
                           pos.stride(0), pos.stride(1), pos.stride(2), rope.table.data_ptr(), rope.table.shape[0],
                           rope.status.data_ptr())
        _lib.call_on(xs[0].device, "ress_rotate", ctypes.addressof(args))
    return ys


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pos, rope, *xs):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(pos)
        ctx.rope, ctx.like = rope, [(x.shape, x.dtype) for x in xs]
        return tuple(_turn(xs, pos, rope, False))

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        pos, = ctx.saved_tensors
        at = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[2 + i]]
        out = [None] * len(grads)
        if at:
            for i, g in zip(at, _turn([grads[i] for i in at], pos, ctx.rope, True)):
                out[i] = g
        return (None, None, *out)


def rotate(x, pos, rope):
    """Rotary positions by a RotaryTable `rope` (its layout, dims, axes and scaling), with a backward pass. x (B, heads, n,
    head_dim) bfloat16 or float16, any strides, or a tuple of two such (queries and keys) of different heads, turned in one
    launch; pos (B, n) or (n,) whole numbers, for two axes (B, n, 2) or (n, 2), on the operands' device. Angles are formed in 64
    bits (RotaryTable), each result is rounded once. Positions outside the table are clamped and reported by rope.check().
    The results are laid out as the operands."""
    xs = [x] if torch.is_tensor(x) else list(x)
    if not 1 <= len(xs) <= 2:
        raise ValueError(f"one or two operands can be turned together, got {len(xs)}")
    first = xs[0]
    for t in xs:
        if not torch.is_tensor(t) or not t.is_cuda:
            raise RuntimeError("x must be a device tensor (the rotation runs only on the GPU)")
        if t.dtype not in DTYPES:
            raise TypeError(f"x must be bfloat16 or float16, got {t.dtype}")
        if t.dim() != 4 or t.shape[3] != rope.head_dim:
            raise ValueError(f"x must be (B, heads, n, {rope.head_dim}), got {tuple(t.shape)}")
        if t.dtype != first.dtype or t.device != first.device or (t.shape[0], t.shape[2]) != (first.shape[0], first.shape[2]):
            raise ValueError("operands that are turned together must have the type, device, batch and tokens of the first")
    B, _, n, _ = first.shape
    if rope.table.device != first.device:
        raise ValueError(f"rope is on {rope.table.device}, x on {first.device}")
    axes = rope.axes
    want = [(B, n), (n,)] if axes == 1 else [(B, n, 2), (n, 2)]
    if not torch.is_tensor(pos) or pos.is_floating_point() or tuple(pos.shape) not in want or pos.device != first.device:
        raise ValueError(f"pos must be {want[0]} or {want[1]} whole numbers on {first.device}")
    pos = pos if pos.dtype is torch.int64 else pos.to(torch.int64)
    pos = pos[..., None] if axes == 1 else pos
    pos = pos if pos.dim() == 3 else pos[None].expand(B, -1, -1)
    if _differentiates(*xs):
        ys = _Rotate.apply(pos, rope, *xs)
    else:
        ys = _turn(xs, pos, rope, False)
    return ys[0] if torch.is_tensor(x) else tuple(ys)
