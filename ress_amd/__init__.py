"""MI355X-native block-sparse global attention for ReSS / HeSS / SparseVGGT.

    import ress_amd as ress
    ress.apply_hess(model, sparse_ratio=0.7)     # model wired with wire_ress_attention
    out = model(images)

Frames that arrive one after the other go through FrameStream, over 8-bit key/value caches; with
quantize_linears the model's linear layers run in 8-bit integers.

The hot path runs on hand-written HIP kernels for gfx950 (libress_hip.so, built by
`python -m ress_amd.build`); see ress_amd.attention for the per-layer pipeline.
"""

from ress_amd.api import apply_dense, apply_hess, apply_ress, apply_sparse_vggt, load_backbone
from ress_amd.attention import check_layers
from ress_amd.backbones import BACKBONES, get_backbone
from ress_amd.int8 import Int8Linear, int8_linear, quantize_linears
from ress_amd.kvcache import PagedKVCache, RotaryTable
from ress_amd.qkv import declare_rope
from ress_amd.stream import FrameStream

__all__ = [
    "BACKBONES",
    "FrameStream",
    "Int8Linear",
    "PagedKVCache",
    "RotaryTable",
    "apply_dense",
    "apply_hess",
    "apply_ress",
    "apply_sparse_vggt",
    "check_layers",
    "declare_rope",
    "get_backbone",
    "int8_linear",
    "load_backbone",
    "quantize_linears",
]
