"""Gradients through a model whose global attention is block-sparse: for fine-tuning under the sparse attention, and for the
gradients that head calibration tables are made of.

    ress.apply_ress(model, ...)            # or any other mode, or none
    ress.enable_gradients(model)
    loss(model(images)).backward()

The package's other operators are made for inference and have no backward pass. Where gradients are asked for, the blocks
of ress_amd.aggregator and every wired attention then run on those of ress_amd.differentiable: layer norms (with the residual
sum and LayerScale in front of them), rotary positions, dense attention, and attention over the selected block map. The map itself
is selected as in inference, by the same kernels, and passes no gradients. Without gradients (torch.no_grad) nothing
changes. The reference has no counterpart: its sparse path runs without gradients, and its calibration through the backbone's
own dense attention (scripts/calibrate_fisher_scores.py).
"""

import torch
import torch.nn as nn

from ress_amd import _lib
from ress_amd.differentiable import (DTYPES, MOST_ROWS, MOST_WIDTH, NORM_DTYPES, Q_BLOCK, _capturing, add_layer_norm,
                                      block_attention, layer_norm, rotate)
from ress_amd.kvcache import RotaryTable
from ress_amd.qkv import grid_shape, rope_base
from ress_amd.stream import POSITIONS

_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")
_GLOBAL_HOOKS = tuple("_global" + h for h in _HOOKS)


def _untouched(module):
    """Whether a call of the module runs its class' forward and nothing else: no hooks, its own or those on every module, and no
    forward put on the instance."""
    return ("forward" not in getattr(module, "__dict__", ()) and not any(getattr(module, h, None) for h in _HOOKS)
            and not any(getattr(nn.modules.module, h, None) for h in _GLOBAL_HOOKS))


def _bare(module, kind):
    """Whether a module is one of `kind` itself and nothing hangs on it, so that its arithmetic can be done in its place."""
    return type(module) is kind and _untouched(module)


def _norm_takes(norm, x):
    if not (_bare(norm, nn.LayerNorm) and len(norm.normalized_shape) == 1 and x.is_cuda and x.dtype in NORM_DTYPES):
        return False
    width = norm.normalized_shape[0]
    kinds = {w.dtype for w in (norm.weight, norm.bias) if w is not None}
    return (x.shape[-1] == width <= MOST_WIDTH and x.numel() <= MOST_ROWS * width and len(kinds) <= 1
            and kinds <= {x.dtype, torch.float32})


def _norm(norm, x):
    return layer_norm(x, norm.weight, norm.bias, norm.eps) if _norm_takes(norm, x) else norm(x)


def _head_norm(norm, x):
    """_norm of queries or keys. Autocast has a norm hand on 32 bits, which the rotation behind it then takes (by the module): nothing is
    rounded between the two."""
    if x.is_cuda and torch.is_autocast_enabled("cuda") and x.dtype is not torch.float32 and _norm_takes(norm, x):
        x = x.float()
    return _norm(norm, x)


def _table(rope, head_dim, device, last):
    """The rotation table of a rotary module of known base (RoPE2D itself or a declared module, with nothing on it) for positions up to
    `last`, made once for each power of two of them and kept on the module (not in its state)."""
    from ress_amd.aggregator import RoPE2D
    known = type(rope) is RoPE2D or not isinstance(rope, RoPE2D) or getattr(rope, "ress_rope", None) is not None
    base = rope_base(rope) if known and _untouched(rope) else None
    if base is None:
        return None
    tables = rope.__dict__.setdefault("_ress_rotary_tables", {})
    positions = max(POSITIONS, 1 << int(last).bit_length())
    key = (head_dim, base, str(device), positions)
    table = tables.get(key)
    if table is None:
        if _capturing():
            raise RuntimeError("run the model once before a graph capture: its rotation tables are made then")
        table = RotaryTable(head_dim, positions, base=base, axes=2, device=device)
        torch.cuda.current_stream(device).synchronize()  # once: other streams, and threads that find it, read it too
        tables[key] = table
    return table


def normed_and_turned(attn, qkv, pos, nh):
    """q, k, v (B, heads, T, head_dim) of a projection's output (B, T, 3 heads head_dim), after the module's q and k norms and its
    rotation, with gradients. Norms and rotary modules that the kernels do not stand for run as they are. Positions that no grid of the
    call's tokens has, and none of a table, are clamped and reported by check_layers."""
    B, T, C = qkv.shape
    hd = C // (3 * nh)
    q, k, v = qkv.reshape(B, T, 3, nh, hd).permute(2, 0, 3, 1, 4).unbind(0)
    q, k = _head_norm(attn.q_norm, q), _head_norm(attn.k_norm, k)
    rope = getattr(attn, "rope", None)
    if rope is not None and pos is not None:
        # a grid its maker has put on the positions, else no side is longer than all tokens
        last = max(getattr(pos, "ress_patch_grid", None) or (T,))
        table = _table(rope, hd, q.device, last) if hd in (64, 128) and q.dtype in (torch.bfloat16, torch.float16) and q.is_cuda else None
        if table is None:
            q, k = rope(q, pos), rope(k, pos)
        else:
            q, k = rotate((q, k), pos.to(q.device), table)
    return q.to(v.dtype), k.to(v.dtype), v


def compute_qkv(self, x, pos, num_special_tokens, num_heads, shape):
    """ress_amd.qkv.compute_qkv with gradients."""
    shp = grid_shape(x, pos, num_special_tokens, num_heads, shape)
    return (*normed_and_turned(self, self.qkv(x), pos, shp["num_heads"]), shp)


class _Gather(torch.autograd.Function):
    """x[..., take, :] of (B, H, T, D); `back`, for each row of x, where it went (every row goes to one place, places may hold copies
    of rows whose gradients are zero)."""

    @staticmethod
    def forward(ctx, x, take, back, pad):
        ctx.save_for_backward(take, back)
        ctx.pad = pad
        return x.index_select(2, take)

    @staticmethod
    def backward(ctx, grad):
        _, back = ctx.saved_tensors
        return grad.index_select(2, back), None, None, None


class _Scatter(torch.autograd.Function):
    """The inverse: rows `back` of o, with zero gradients for the places in `pad`, which hold copies."""

    @staticmethod
    def forward(ctx, o, take, back, pad):
        ctx.save_for_backward(take)
        ctx.pad = pad
        return o.index_select(2, back)

    @staticmethod
    def backward(ctx, grad):
        take, = ctx.saved_tensors
        g = grad.index_select(2, take)
        lo, hi = ctx.pad
        if hi > lo:
            g[:, :, lo:hi] = 0
        return g, None, None, None


def _orders(grid, patch_order, device):
    """Index tensors of a layer's blocks, in storage order's terms: (keys, back of keys, queries, back of queries, pad).
    Keys are the patch tokens (in the blocks' order), then the special ones; queries the same with the patch tokens filled up to
    whole blocks of 128 in between."""
    P, S, N = grid.P, grid.S, grid.frames
    hw = P - S
    within = torch.arange(hw, device=device) if patch_order is None else patch_order.to(device=device, dtype=torch.int64)
    frame = torch.arange(N, device=device)[:, None] * P
    patch = (frame + S + within[None]).reshape(-1)
    special = (frame + torch.arange(S, device=device)[None]).reshape(-1)
    keys = torch.cat([patch, special])
    fill = -len(patch) % Q_BLOCK if S else 0
    queries = torch.cat([patch, patch.new_zeros(fill), special])
    at = torch.arange(N * P, device=device)
    k_back = torch.empty_like(at).scatter_(0, keys, at)
    place = torch.cat([at[: len(patch)], at[len(patch):] + fill])
    q_back = torch.empty_like(at).scatter_(0, keys, place)
    return keys, k_back, queries, q_back, (len(patch), len(patch) + fill)


_plain_orders = {}  # (frames, tokens a frame, special ones, device, stream) -> _orders without a patch order


def _layer_orders(grid, patch_order, device):
    if patch_order is not None or _capturing():  # what is made inside a capture belongs to its graph
        return _orders(grid, patch_order, device)
    key = (grid.frames, grid.P, grid.S, str(device), _lib.stream_handle(device))
    orders = _plain_orders.get(key)  # by itself: other threads put tables in and clear them
    if orders is None:
        orders = _orders(grid, None, device)
        if len(_plain_orders) >= 8:
            _plain_orders.clear()
        _plain_orders[key] = orders
    return orders


def sparse_attention(q, k, v, final_map, grid, patch_order=None):
    """The attention of a block-sparse layer over its map, with gradients: q, k, v (B, H, frames P, head_dim) in storage order; patch
    queries see the blocks of final_map (B, H, q blocks, key blocks), special ones everything."""
    keys, k_back, queries, q_back, pad = _layer_orders(grid, patch_order, q.device)
    none = (0, 0)
    qo = _Gather.apply(q, queries, q_back, pad)
    ko, vo = _Gather.apply(k, keys, k_back, none), _Gather.apply(v, keys, k_back, none)
    m = final_map.to(torch.bool)
    blocks = -(-len(queries) // Q_BLOCK) - m.shape[2]  # of special queries
    if blocks:
        m = torch.cat([m, m.new_ones(*m.shape[:2], blocks, m.shape[3])], 2)
    out = block_attention(qo, ko, vo, block_map=m)
    return _Scatter.apply(out, queries, q_back, pad)


def attention_forward(attn, x, pos=None):
    """ress_amd.aggregator.Attention's forward with gradients."""
    B, T, C = x.shape
    nh = attn.num_heads
    q, k, v = normed_and_turned(attn, attn.qkv(x), pos, nh)
    o = block_attention(q, k, v)
    return attn.proj_drop(attn.proj(o.transpose(1, 2).reshape(B, T, C)))


def block_forward(block, x, pos=None):
    """ress_amd.aggregator.Block's forward with gradients: the residual sum behind the attention and the norm behind it are one operator
    where nothing hangs on the modules."""
    from ress_amd.aggregator import LayerScale
    a = block.attn(_norm(block.norm1, x), pos=pos)
    ls, norm = block.ls1, block.norm2
    if (_bare(ls, LayerScale) and _norm_takes(norm, x) and a.dtype == x.dtype
            and all(w is None or w.dtype == ls.gamma.dtype for w in (norm.weight, norm.bias)) and ls.gamma.dtype in (x.dtype, torch.float32)):
        x, n = add_layer_norm(x, a, ls.gamma, norm.weight, norm.bias, norm.eps)
    else:
        x = x + ls(a)
        n = _norm(norm, x)
    return x + block.ls2(block.mlp(n))


def enable_gradients(model, on=True):
    """Has the model's blocks (those of ress_amd.aggregator) and its wired attentions run on operators with a backward pass wherever
    gradients are asked for, on the GPU in 16 bits (a 32-bit model under autocast, or wired: its sparse layers run in bfloat16, its dense
    ones by torch in 32 bits). Heads of 64 or 128. on=False takes it back. Returns the model."""
    from ress_amd.aggregator import Attention, Block
    from ress_amd.wiring import SparseAttentionForward
    found = []
    for module in model.modules():
        wired = isinstance(getattr(module, "forward", None), SparseAttentionForward)
        if isinstance(module, Attention):
            hd = module.qkv.in_features // module.num_heads
            if hd not in (64, 128) and not wired:
                raise ValueError(f"the attention with gradients takes heads of 64 or 128, got {hd}")
        if wired or isinstance(module, (Attention, Block)):
            found.append((module, wired))
    if not found:
        raise TypeError(f"{type(model).__name__} has neither blocks of ress_amd.aggregator nor wired attentions")
    for module, wired in found:
        if wired:
            module.differentiable = bool(on)
        if isinstance(module, (Attention, Block)):
            module.gradients = bool(on)
    return model
