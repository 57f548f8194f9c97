"""Operators with a backward pass: what a block of the model runs in a training or calibration step.

    out = block_attention(q, k, v, block_map=kept)            # softmax attention over a map of 128-query x 64-key blocks
    h, n = add_layer_norm(x, branch, gamma, weight, bias)     # x + gamma * branch, and its layer norm
    q, k = rotate((q, k), pos, rope)                          # rotary positions by a RotaryTable

The block-sparse layers run without gradients. Calibration tables (a head's Fisher scores) and fine-tuning under a fixed
map need them; ress_amd.training puts these operators into a model's blocks.

Every operator works on torch's current stream of its operands' device, waits for nothing and repeats bit for bit: no sum
is made by atomics. Gradients are formed once (no second derivatives, none in forward mode: dual tensors are refused), in the
operands' types with 32-bit sums.
Operands with strides that a kernel cannot take are copied first. The reference has no counterpart: its kernels have no
backward pass.

In a captured graph: torch accumulates a leaf's gradient on the stream on which the leaf entered the oldest graph that still
lives. Where that is an eager one of the default stream, capturing the backward pass would end the process: a call with a leaf
of which these operators have made such a graph is refused inside a capture (delete the eager result first, or run it on a side stream;
graphs that torch's operators alone have made of a leaf cannot be told).
"""

import functools
import math
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ress_amd import _lib

DTYPES = {torch.bfloat16: 1, torch.float16: 2}
Q_BLOCK, K_BLOCK = 128, 64
MOST_TOKENS, MOST_MAPPED = 1 << 26, 1 << 20
MOST_STRIDE = 1 << 24

# The argument structs of include/ress_hip.h, packed (a call's host time is what a small one costs).
_STRIDED = struct.Struct("@4q").pack           # ress_strided, ress_rows: data and three strides
_ATTN = struct.Struct("@16q8i3q4q2qf4x").pack   # ress_block_attn
_NORM = struct.Struct("@8q6i7qf4x").pack        # ress_layer_norm
_ROTARY = struct.Struct("@16q10i5qi4xq").pack   # ress_rotary


def _capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _differentiates(*tensors):
    """Whether a call on these tensors makes a graph; refuses tangents, and leaves whose gradients cannot be captured."""
    if forward_ad._current_level >= 0:  # inside a dual level, with gradients or without
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the operators have a backward pass but no forward-mode derivatives (a dual tensor was given)")
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            break
    else:
        return False
    if torch.cuda.is_current_stream_capturing():
        for t in tensors:
            if t is not None and t.requires_grad and t.is_leaf:
                if "ress_default_stream" in torch.autograd.graph.get_gradient_edge(t).node.metadata:
                    raise RuntimeError("inside a graph capture: a result of the same leaves from outside of it, on the "
                                       "default stream, is still alive; delete it first")
    return True


def _mark(result, device):
    """Notes at the leaves of a graph that was made on the default stream that it was (the note lives as long as a graph
    with the leaf does)."""
    if not _lib.stream_handle(device):
        for node, _ in result.grad_fn.next_functions:
            if node is not None and node.name() == "torch::autograd::AccumulateGrad":
                node.metadata["ress_default_stream"] = True


def _first_derivative(function):
    """A backward function that makes no graph of its own; torch's guard only where one is asked for."""
    guarded = once_differentiable(function)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else function(ctx, *grads)
    return staticmethod(backward)


def _empty(t):
    """A contiguous tensor like t (empty_like takes a third of empty's host time)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


# ---- attention -------------------------------------------------------------------
def _strides(t):
    """(address, batch, heads, tokens) of t (B, H, T, D) as the kernels take it, strides of single entries in their place;
    None where they cannot."""
    B, H, T, D = t.shape
    sb, sh, st, sd = t.stride()
    if B == 1:
        sb = 0
    if H == 1:
        sh = 0
    if T == 1:
        st = D
    at = t.data_ptr()
    if sd != 1 or st < D or st >= MOST_STRIDE or (sb | sh | st) & 7 or at & 15:
        return None if t.numel() else (at, 0, 0, D)
    return at, sb, sh, st


def _ready(t):
    """(t or a copy that the kernels can take, its _strides)"""
    at = _strides(t)
    if at is None:
        t = t.clone(memory_format=torch.contiguous_format)
        at = _strides(t)
    return t, at


def _like(t):
    """(a tensor for a result laid out like t where the kernels can write that, its _strides)"""
    new = torch.empty_like(t)
    at = _strides(new)
    if at is None:
        new = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        at = _strides(new)
    return new, at


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


def _attn_args(q, k, at, block_map, causal, q_lens, k_lens, scale, lse, rest):
    """at: the _strides of q, k, v and the output, one behind the other"""
    B, Hq, Tq, D = q.shape
    if block_map is None:
        m = (0, 0, 0, 0, 0)
    else:
        m = (block_map.data_ptr(), *block_map.stride())
    return _ATTN(*at, B, Hq, k.shape[1], Tq, k.shape[2], D, DTYPES[q.dtype],
                 1 if causal else 0, 0 if q_lens is None else q_lens.data_ptr(), 0 if k_lens is None else k_lens.data_ptr(), *m,
                 0 if lse is None else lse.data_ptr(), 0 if rest is None else rest.data_ptr(), scale)


def _attend(q, k, v, block_map, causal, q_lens, k_lens, scale, grads):
    """q, k, v: what _ready gave for them"""
    (q, aq), (k, ak), (v, av) = q, k, v
    out, ao = _like(q)
    lse = rest = None
    if grads:
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
        rest = _empty(q)
    if out.numel():
        args = _attn_args(q, k, aq + ak + av + ao, block_map, causal, q_lens, k_lens, scale, lse, rest)
        size, work = _attn_workspace(False, args[128:160], block_map is not None), None
        if size:
            work = torch.empty(size, dtype=torch.uint8, device=q.device)
        _lib.call_on(q.device, "ress_block_attn_fwd", args, None if work is None else work.data_ptr(), size)
    return out, lse, rest


class _BlockAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, block_map, causal, q_lens, k_lens, scale):
        q, k, v = _ready(q), _ready(k), _ready(v)
        out, lse, rest = _attend(q, k, v, block_map, causal, q_lens, k_lens, scale, True)
        ctx.save_for_backward(q[0], k[0], v[0], out, lse, rest, block_map, q_lens, k_lens)
        ctx.how = causal, scale
        return out

    @_first_derivative
    def backward(ctx, grad):
        q, k, v, out, lse, rest, block_map, q_lens, k_lens = ctx.saved_tensors
        causal, scale = ctx.how
        grad, ag = _ready(grad)
        (dq, aq), (dk, ak), (dv, av) = _like(q), _like(k), _like(v)
        args = _attn_args(q, k, _strides(q) + _strides(k) + _strides(v) + _strides(out), block_map, causal, q_lens, k_lens, scale,
                          lse, rest)
        size = _attn_workspace(True, args[128:160], block_map is not None)
        work = torch.empty(size, dtype=torch.uint8, device=q.device)
        _lib.call_on(q.device, "ress_block_attn_bwd", args, _STRIDED(*ag), _STRIDED(*aq), _STRIDED(*ak), _STRIDED(*av),
                     work.data_ptr(), size)
        return dq, dk, dv, None, None, None, None, None


@functools.lru_cache(maxsize=256)
def _attn_workspace(backward, sizes, mapped):
    size = _lib.lib().ress_block_attn_bwd_workspace_size if backward else _lib.lib().ress_block_attn_fwd_workspace_size
    return size(bytes(128) + sizes + struct.pack("@3q", 0, 0, 1 if mapped else 0) + bytes(64))


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
    hold; a key or value that is not finite makes NaN of the rows that see its block, in causal order also of the others of
    their 128-query blocks.

    The probabilities, formed anew in the backward pass, and the scores' gradients are rounded to the operands' type before
    they are multiplied; half of the latter, for dq, and both in calls of up to 2^18 probabilities (all sequences and heads,
    whatever a map or the causal order leaves), are multiplied in two terms. Sums, maxima and the softmax's statistics are
    fp32. A forward pass for gradients keeps, beside its operands and output, a tensor of the output's size (what its
    rounding took) and 4 bytes a row."""
    _check_attention(q, k, v, block_map)
    B, Hq, Tq, D = q.shape
    if torch.is_tensor(scale) and scale.requires_grad and torch.is_grad_enabled():
        raise ValueError("scale gets no gradient: give a number, and multiply q by what is learnt")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if q_lens is not None:
        q_lens = _lens(q_lens, "q_lens", B, Tq, q.device)
    if k_lens is not None:
        k_lens = _lens(k_lens, "k_lens", B, k.shape[2], q.device)
    if block_map is not None:
        block_map = block_map.expand(B, Hq, -1, -1)
    if _differentiates(q, k, v):
        out = _BlockAttention.apply(q, k, v, block_map, causal, q_lens, k_lens, scale)
        _mark(out, q.device)
        return out
    return _attend(_ready(q), _ready(k), _ready(v), block_map, causal, q_lens, k_lens, scale, False)[0]


# ---- layer norm ------------------------------------------------------------------
NORM_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST_WIDTH, MOST_ROWS = 8192, (1 << 31) - 1


def _rows(tensors):
    """((n0, n1, n2), operands): the rows (..., C) of tensors of one shape (None stays), each as (address, three strides, tensor);
    those whose rows the kernels cannot take are copied."""
    first = tensors[0]
    C = first.shape[-1]
    for t in tensors:
        if t is not None and not t.is_contiguous():
            break
    else:
        return (first.numel() // C, 1, 1), [(0, 0, 0, 0, None) if t is None else (t.data_ptr(), C, 0, 0, t) for t in tensors]
    shape = first.shape
    lead = [i for i in range(len(shape) - 1) if shape[i] > 1]
    if len(lead) > 3:
        return _rows([t if t is None else t.contiguous() for t in tensors])
    tensors = [t if t is None or t.stride(-1) == 1 or C == 1 else t.contiguous() for t in tensors]
    pad = [None] * (3 - len(lead))
    axes = lead + pad if len(lead) == 1 else pad + lead  # one axis goes first: its rows are found without a division

    def row(t):
        return (0, 0, 0, 0, None) if t is None else (t.data_ptr(), *(0 if i is None else t.stride(i) for i in axes), t)

    return tuple(1 if i is None else shape[i] for i in axes), [row(t) for t in tensors]


def _normalise(x, branch, gamma, weight, bias, eps, grads):
    """(sum or None, n, mean and rstd or None)"""
    sizes, (xr, br) = _rows((x, branch))
    out = _empty(x)
    total = _empty(x) if branch is not None else None
    stats = torch.empty((2, sizes[0] * sizes[1] * sizes[2]), dtype=torch.float32, device=x.device) if grads else None
    if out.numel():
        at = stats.data_ptr() if grads else 0
        w = gamma if gamma is not None else weight if weight is not None else bias
        args = _NORM(*xr[:4], *br[:4], *sizes, x.shape[-1], NORM_DTYPES[x.dtype],
                     1 if w is not None and w.dtype is torch.float32 else 0, 0 if gamma is None else gamma.data_ptr(),
                     0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
                     0 if total is None else total.data_ptr(), out.data_ptr(), at, at + 2 * stats.numel() if grads else 0, eps)
        _lib.call_on(x.device, "ress_layer_norm_fwd", args)
    return total, out, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gamma, weight, bias, eps):
        ctx.set_materialize_grads(False)
        total, out, stats = _normalise(x, branch, gamma, weight, bias, eps, True)
        ctx.save_for_backward(x if branch is None else total, branch, gamma, weight, bias, stats)
        ctx.eps = eps
        return out if branch is None else (total, out)

    @_first_derivative
    def backward(ctx, *grads):
        h, branch, gamma, weight, bias, stats = ctx.saved_tensors
        to_x, to_branch, to_gamma, to_weight, to_bias, _ = ctx.needs_input_grad
        dn = grads[-1]
        dh = grads[0] if branch is not None else None
        if dh is None and dn is None:
            return None, None, None, None, None, None
        dx = _empty(h) if to_x or (to_branch and gamma is None) else None
        dbranch = _empty(h) if to_branch and gamma is not None else None
        dgamma = _empty(gamma) if to_gamma else None
        dweight = _empty(weight) if to_weight else None
        dbias = _empty(bias) if to_bias else None
        if h.numel() == 0:
            for t in (dgamma, dweight, dbias):
                if t is not None:
                    t.zero_()
        else:
            sizes, (hr, br, nr, sr) = _rows((h, branch, dn, dh))
            w = gamma if gamma is not None else weight if weight is not None else bias
            at = stats.data_ptr()
            args = _NORM(*hr[:4], *br[:4], *sizes, h.shape[-1], NORM_DTYPES[h.dtype],
                         1 if w is not None and w.dtype is torch.float32 else 0, 0 if gamma is None else gamma.data_ptr(),
                         0 if weight is None else weight.data_ptr(), 0, 0, 0, at, at + 2 * stats.numel(), ctx.eps)
            size, work = 0, None
            if to_gamma or to_weight or to_bias:
                size = _norm_workspace(args[64:88])
                work = torch.empty(size, dtype=torch.uint8, device=h.device)
            _lib.call_on(h.device, "ress_layer_norm_bwd", args, None if dn is None else _STRIDED(*nr[:4]),
                         None if dh is None else _STRIDED(*sr[:4]), None if dx is None else dx.data_ptr(),
                         None if dbranch is None else dbranch.data_ptr(), None if dgamma is None else dgamma.data_ptr(),
                         None if dweight is None else dweight.data_ptr(), None if dbias is None else dbias.data_ptr(),
                         None if work is None else work.data_ptr(), size)
        if to_branch and gamma is None:
            dbranch = dx
        return dx if to_x else None, dbranch, dgamma, dweight, dbias, None


@functools.lru_cache(maxsize=256)
def _norm_workspace(sizes):
    return _lib.lib().ress_layer_norm_bwd_workspace_size(bytes(64) + sizes + bytes(64))


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
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if _differentiates(x, weight, bias):
        n = _LayerNorm.apply(x, None, None, weight, bias, eps)
        _mark(n, x.device)
        return n
    return _normalise(x, None, None, weight, bias, eps, False)[1]


def add_layer_norm(x, branch, gamma=None, weight=None, bias=None, eps=1e-5):
    """(h, n): the residual sum h = x + gamma * branch and n = layer_norm(h, weight, bias, eps), in one pass over x and branch and with
    one backward pass, to all five. branch: shape and type of x; gamma (a LayerScale), weight, bias: (C,), of x's type or, all of
    them, float32 (None: 1, 1 and 0). The norm is that of h as it is returned, rounded to its type."""
    eps = float(eps)
    if branch is None:
        raise ValueError("branch is missing (layer_norm takes x alone)")
    _check_norm(x, branch, gamma, weight, bias, eps)
    gamma, weight, bias = (t if t is None or t.is_contiguous() else t.contiguous() for t in (gamma, weight, bias))
    if _differentiates(x, branch, gamma, weight, bias):
        both = _LayerNorm.apply(x, branch, gamma, weight, bias, eps)
        _mark(both[0], x.device)
        return both
    return _normalise(x, branch, gamma, weight, bias, eps, False)[:2]


# ---- rotary positions ------------------------------------------------------------
def _turn(xs, pos, rope, inverse):
    """The operands turned (one or two), each in a tensor laid out like it."""
    xs = [x if x.stride(3) == 1 else x.contiguous() for x in xs]
    ys = [torch.empty_like(x) for x in xs]
    ys = [y if y.stride(3) == 1 else _empty(y) for y in ys]
    x, y = xs[0], ys[0]
    B, H, n, D = x.shape
    if n and B:
        x2 = y2 = (0, 0, 0, 0)
        H2 = 0
        if len(xs) > 1:
            x2, y2 = (xs[1].data_ptr(), *xs[1].stride()[:3]), (ys[1].data_ptr(), *ys[1].stride()[:3])
            H2 = xs[1].shape[1]
        args = _ROTARY(x.data_ptr(), *x.stride()[:3], *x2, y.data_ptr(), *y.stride()[:3], *y2, H, H2, B, n, D, DTYPES[x.dtype],
                       rope.axes, rope.rotary_dim, 1 if rope.layout == "interleaved" else 0, 1 if inverse else 0, pos.data_ptr(),
                       *pos.stride(), rope.table.data_ptr(), rope.table.shape[0], rope.status.data_ptr())
        _lib.call_on(x.device, "ress_rotate", args)
    return ys


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pos, rope, *xs):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(pos)
        ctx.rope = rope
        return tuple(_turn(xs, pos, rope, False))

    @_first_derivative
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
    if rope.table.requires_grad and torch.is_grad_enabled():
        raise ValueError("the rotation table gets no gradient: give one that does not require it")
    axes = rope.axes
    want = [(B, n), (n,)] if axes == 1 else [(B, n, 2), (n, 2)]
    if not torch.is_tensor(pos) or pos.is_floating_point() or tuple(pos.shape) not in want or pos.device != first.device:
        raise ValueError(f"pos must be {want[0]} or {want[1]} whole numbers on {first.device}")
    pos = pos if pos.dtype is torch.int64 else pos.to(torch.int64)
    pos = pos[..., None] if axes == 1 else pos
    pos = pos if pos.dim() == 3 else pos[None].expand(B, -1, -1)
    if _differentiates(*xs):
        ys = _Rotate.apply(pos, rope, *xs)
        _mark(ys[0], first.device)
    else:
        ys = _turn(xs, pos, rope, False)
    return ys[0] if torch.is_tensor(x) else tuple(ys)
