"""Attention over long caches whose keys are split into parts: the join by whole rows (from 2,048 rows on) and by
workgroups a row, ragged and padded batches, and more parts than a join's lanes weigh at once. Against 64 bits."""

import ctypes

import pytest
import torch

from kvcache_oracle import attention, held, tolerance
from ress_amd import _lib
from ress_amd.kvcache import PAGE, PagedKVCache, _CacheArgs

BF16, F16 = torch.bfloat16, torch.float16

# name: (query heads a head, heads, rows, head dim, lengths, new tokens or None, parts that the longest is cut into at least)
CASES = {
    "ragged": (1, 2, 400, 64, [9000, 700, 0, 4100], None, 16),
    "ragged padded": (1, 2, 400, 64, [9000, 700, 0, 4100], [400, 399, 7, 0], 16),
    "ragged grouped 128": (4, 1, 200, 128, [6000, 100, 3000], None, 8),
    "padded 128": (1, 3, 400, 128, [6000, 5000], [400, 130], 8),
    "more parts than lanes": (1, 2, 1100, 64, [20000], None, 17),
    "many rows 128": (1, 1, 2100, 128, [20000], None, 25),
    "a row over a long cache": (1, 1, 1, 64, [240000], None, 257),
    "a row over a long cache 128": (1, 1, 1, 128, [240000], None, 257),
    "few rows, ragged": (2, 1, 3, 64, [150000, 300, 0, 70000], [3, 1, 2, 0], 60),
}


def _parts(G, H, n, D, B, longest):
    c = _CacheArgs(*[4096] * 12, 8192, 8192, B, H, D, 1, 0)
    size = _lib.lib().ress_kv_attend_workspace_size(ctypes.addressof(c), B, G * H, n, longest)
    return size // (4 * B * G * H * n * (D + 2))


@pytest.mark.parametrize("name", CASES)
def test_parts(name):
    G, H, n, D, lens, _, least = CASES[name]
    assert _parts(G, H, n, D, len(lens), max(lens)) >= least
    wide = len(lens) * G * H * n >= 2048
    lanes = D // 4 * (1 if wide else 256 // (D // 4))  # parts that a row's lanes weigh at once
    assert ("more parts" in name or "long cache" in name) == (least > lanes)
    assert wide == (n >= 200)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,codes", [(BF16, "int8"), (F16, "fp8"), (BF16, "fp8"), (F16, "int8")])
@pytest.mark.parametrize("name", CASES)
def test_joined_rows(dev, dtype, codes, name):
    G, H, n, D, lens, news, _ = CASES[name]
    B, T = len(lens), max(lens)
    g = torch.Generator(device=dev).manual_seed(len(name))

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    pages = sum(-(-(L + 1) // PAGE) for L in lens)
    c = PagedKVCache(pages, H, D, max_seqs=B, max_len=T + 1, dtype=dtype, codes=codes, device=dev)
    off = rand(2, 1, H, 1, D)
    for b, L in enumerate(lens):
        if L:
            c.append(*((rand(1, H, L, D) + o).to(dtype) for o in off), slots=[b])
    q = (rand(B, G * H, n, D) * 1.5).to(dtype)
    assert c.lengths() == lens and max(c._bound) == T  # so the call is cut as test_parts says
    for causal in (False, True):
        got = c.attend(q, causal=causal, new_lens=news)
        out = torch.full_like(q, 5.0)
        assert c.attend(q, causal=causal, new_lens=news, out=out) is out
        for b, L in enumerate(lens):
            m = n if news is None else news[b]
            assert (got[b, :, m:] == 0).all() and (out[b, :, m:] == 5).all() and torch.equal(got[b, :, :m], out[b, :, :m])
            if L == 0:
                assert (got[b] == 0).all()
                continue
            k, v = held(c, b)
            rows = sorted({i for i in (0, 1, 15, 16, 31, 32, 63, 127, 128, 255, 256, n // 2, m - 3, m - 2, m - 1) if 0 <= i < m})
            for i in rows:
                seen = min(L, max(0, L - m + i + 1)) if causal else L
                row = got[b, :, i:i + 1]
                if seen == 0:
                    assert (row == 0).all()
                    continue
                want, size, spread = attention(q[b, :, i:i + 1], k[:, :seen], v[:, :seen], 1, False)
                err = (row.double().cpu() - want).abs()
                tol = tolerance(want, size, spread, dtype, seen)
                assert (err <= tol).all(), (b, i, causal, float((err / tol).max()))
    c.check()
