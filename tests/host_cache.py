"""A PagedKVCache without a GPU: its host side on CPU tensors, the append kernel's effect on lengths restated."""

import contextlib

import torch

from ress_amd import kvcache
from ress_amd.kvcache import PAGE, PagedKVCache


def host_cache(monkeypatch, n_pages=8, max_seqs=2, max_pages=None, fail=None):
    """fail: a dict whose "append", once set, is raised by the library call instead."""
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(kvcache._lib, "ptr", lambda t: t)
    c = PagedKVCache.__new__(PagedKVCache)
    c.device, c.dtype, c.codes = torch.device("cpu"), torch.bfloat16, "int8"
    c.n_pages, c.kv_heads, c.head_dim, c.max_seqs = n_pages, 1, 64, max_seqs
    c.max_pages = max_pages or n_pages
    c._state = torch.zeros(4 * max_seqs, dtype=torch.uint8)
    c.lens = c._state.view(torch.int32)
    c.table = torch.full((max_seqs, c.max_pages), -1, dtype=torch.int32)
    c.held = torch.zeros(max_seqs, dtype=torch.int32)
    c._status = torch.zeros(1, dtype=torch.int32)
    c._free = list(range(n_pages - 1, -1, -1))
    c._pages = [[] for _ in range(max_seqs)]
    c._bound, c._cap = [0] * max_seqs, [0] * max_seqs
    c._key, c._lag, c._slack, c._most = None, 0, 0, 0
    c._captured = c._guessed = False
    c._snapshots, c._serial = kvcache.weakref.WeakSet(), 0
    c._handle = None

    def call(name, handle, k, *rest):
        if fail and fail.get("append"):
            raise fail["append"]
        slots, new_lens = rest[-3], rest[-2]
        B, n = k.shape[0], k.shape[2]
        for b in range(B):
            s = b if slots is None else int(slots[b])
            want = int(c.lens[s]) + (n if new_lens is None else min(max(int(new_lens[b]), 0), n))
            room = PAGE * int(c.held[s])
            c.lens[s] = min(want, room)
            if want > room:
                c._status |= 1

    c._call = call
    return c


def tokens(B, n):
    return torch.zeros(B, 1, n, 64, dtype=torch.bfloat16)
