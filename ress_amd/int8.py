"""Linear layers in 8-bit integers: weights held as int8 codes with a scale for each output channel,
activations quantised per token on the way in, products summed exactly in int32.

    quantize_linears(model)          # every suitable nn.Linear becomes an Int8Linear
    y = int8_linear(x, codes, scale, bias, act="gelu")

Half the bytes of 16-bit weights, which is what a call of a few tokens costs, and the matrix cores' 8-bit
rate for many. The reference's layers are torch's 16-bit ones; nothing here is used unless asked for.
"""

import functools

import torch
import torch.nn as nn
from torch.nn.utils import prune
from torch.nn.utils.spectral_norm import SpectralNorm
from torch.nn.utils.weight_norm import WeightNorm

from ress_amd import _lib

DTYPES = {torch.bfloat16: 1, torch.float16: 2}
ACTS = {None: 0, "gelu": 1}
MOST_ROWS = 1 << 30
MOST_FEATURES = 131072  # |sum| <= 127^2 * 131072 < 2^31


def _rows(x, name):
    if not torch.is_tensor(x) or not x.is_cuda:
        raise RuntimeError(f"{name} must be a device tensor (the 8-bit product runs only on the GPU)")
    if x.dtype not in DTYPES:
        raise TypeError(f"{name} must be bfloat16 or float16, got {x.dtype} (cast the model, or run it under autocast)")
    if x.dim() < 1 or x.shape[-1] % 16 or not 0 < x.shape[-1] <= MOST_FEATURES:
        raise ValueError(f"{name} must have a last dim that is a multiple of 16 up to {MOST_FEATURES}, got {tuple(x.shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires grad: the 8-bit product has no backward pass (use torch.no_grad())")
    if x.numel() > MOST_ROWS * x.shape[-1]:
        raise ValueError(f"{name} must have at most {MOST_ROWS} rows, got {tuple(x.shape)}")
    rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if rows.stride(1) != 1 or (len(rows) > 1 and rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()
    return rows


def quantize_tokens(x):
    """(codes int8, scale float32) of x (..., K), bfloat16 or float16, a scale for each row: code =
    round(x * 127 / max|x|) (ties to even), scale = max|x| / 127. A row with an element that is not finite has
    scale NaN and codes 0."""
    rows = _rows(x, "x")
    codes = torch.empty(rows.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(len(rows), dtype=torch.float32, device=x.device)
    _lib.call_on(x.device, "ress_quantize_rows", _lib.ptr(rows), rows.stride(0), DTYPES[x.dtype], len(rows),
                 rows.shape[1], _lib.ptr(codes), rows.shape[1], _lib.ptr(scale))
    return codes.reshape(x.shape), scale.reshape(x.shape[:-1])


def quantize_weight(weight):
    """(codes int8 (N, K), scale float32 (N,)) of a weight matrix of any floating type, once per model."""
    if weight.dim() != 2 or weight.shape[1] % 16 or not 0 < weight.shape[1] <= MOST_FEATURES:
        raise ValueError(f"weight must be (N, K) with K a multiple of 16 up to {MOST_FEATURES}, got {tuple(weight.shape)}")
    w = weight.detach().float()
    if not torch.isfinite(w).all():
        raise ValueError("weight has values that are not finite")
    scale = w.abs().amax(1) / 127.0
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(w / safe[:, None]).clamp(-127, 127).to(torch.int8).contiguous(), scale


def int8_linear(x, w_codes, w_scale, bias=None, act=None):
    """act(x W^T + bias) in x's type, (..., N): x (..., K) bfloat16 or float16, quantised per token as by
    quantize_tokens; W = w_codes (N, K) int8 * w_scale (N,) float32; bias (N,) float32; act None or "gelu" (erf)."""
    rows = _rows(x, "x")
    M, K = rows.shape
    dev = x.device
    if (w_codes.dtype is not torch.int8 or w_codes.dim() != 2 or w_codes.shape[1] != K or not w_codes.is_contiguous()):
        raise ValueError(f"w_codes must be contiguous int8 (N, {K}), got {tuple(w_codes.shape)} {w_codes.dtype}")
    N = w_codes.shape[0]
    for name, t in (("w_scale", w_scale), ("bias", bias)):
        if t is not None and (t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != N or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 ({N},), got {tuple(t.shape)} {t.dtype}")
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires grad: the 8-bit product has no backward pass (use torch.no_grad())")
    if w_codes.device != dev or w_scale.device != dev or (bias is not None and bias.device != dev):
        raise ValueError(f"the weights are not on {dev}")
    if act not in ACTS:
        raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
    out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=dev)
    if M == 0 or N == 0:
        return out
    size = _workspace(M, K, N)
    work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    P = _lib.ptr
    _lib.call_on(dev, "ress_int8_linear", P(rows), rows.stride(0), DTYPES[x.dtype], M, K, N, P(w_codes), P(w_scale),
                 P(bias), ACTS[act], P(out), N, P(work), size)
    return out


@functools.lru_cache(maxsize=256)
def _workspace(M, K, N):
    return _lib.lib().ress_int8_linear_workspace_size(M, K, N)


# what torch's reparametrisations and pruning leave on a layer, which forms the weight anew before each forward
_WEIGHT_HOOKS = (WeightNorm, SpectralNorm, prune.BasePruningMethod)


class Int8Linear(nn.Module):
    """An nn.Linear's place-holder with 8-bit weights (buffers, not parameters), for 16-bit activations; under autocast
    they are cast to its type, as the layer's would be."""

    def __init__(self, linear):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.dtype = linear.weight.dtype
        codes, scale = quantize_weight(linear.weight)
        self.register_buffer("codes", codes)
        self.register_buffer("scale", scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float().contiguous())
        # The layer's mode and forward hooks go with it (the same dicts, so that the hooks' handles still remove them), but for
        # hooks that form its weight, for which the codes stand.
        self.training = linear.training
        for name in ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks",
                     "_forward_pre_hooks_with_kwargs"):
            setattr(self, name, getattr(linear, name))
        if any(isinstance(h, _WEIGHT_HOOKS) for h in self._forward_pre_hooks.values()):
            self._forward_pre_hooks = type(self._forward_pre_hooks)(
                (i, h) for i, h in self._forward_pre_hooks.items() if not isinstance(h, _WEIGHT_HOOKS))

    def _apply(self, fn, recurse=True):
        # a cast of the model to 16 bits must not round the scales and the bias, which are fp32
        kept = {n: getattr(self, n) for n in ("scale", "bias") if getattr(self, n) is not None}
        super()._apply(fn, recurse)
        for n, t in kept.items():
            setattr(self, n, t.to(self.codes.device))
        self.dtype = fn(torch.empty(0, dtype=self.dtype, device=self.codes.device)).dtype
        return self

    @property
    def weight(self):
        """The weights that the codes stand for, in the type that the layer's own would have now."""
        return (self.codes.float() * self.scale[:, None]).to(self.dtype)

    def forward(self, x, act=None):
        if torch.is_autocast_enabled(x.device.type) and x.is_floating_point() and x.dtype is not torch.float64:
            x = x.to(torch.get_autocast_dtype(x.device.type))
        return int8_linear(x, self.codes, self.scale, self.bias, act)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def quantize_linears(model, keep=lambda name, linear: False):
    """Replaces every nn.Linear of the model by an Int8Linear, in place, but for those whose in_features are
    not a multiple of 16 and those that keep(name, linear) names (a layer with several names: by any of them).
    The layers then take 16-bit activations: a 32-bit model is to be cast (before or after) or run under autocast.
    Returns the names replaced. A weight that is not finite is refused before any layer is replaced."""
    places = {}  # linear -> (module, child, full name) of each of its places
    for name, module in model.named_modules():
        for child, linear in module._modules.items():
            if type(linear) is nn.Linear and linear.in_features % 16 == 0 and 0 < linear.in_features <= MOST_FEATURES:
                places.setdefault(linear, []).append((module, child, f"{name}.{child}" if name else child))
    places = {linear: at for linear, at in places.items() if not any(keep(full, linear) for _, _, full in at)}
    for linear, at in places.items():
        if not torch.isfinite(linear.weight).all():
            raise ValueError(f"{at[0][2]}: weight has values that are not finite")
    done = []
    for linear, at in places.items():
        new = Int8Linear(linear)
        for module, child, full in at:
            setattr(module, child, new)
            done.append(full)
    return done
