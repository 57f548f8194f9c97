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
