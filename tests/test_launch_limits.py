"""Calls too large for one launch: a launch counts its threads in 32 bits. Without a GPU: what is refused is refused
before any pointer is used."""

import ctypes

import pytest

from ress_amd import _lib
from ress_amd.kvcache import _CacheArgs

P = ctypes.c_void_p(4096)
F = (P, 0, 0, 64)
Z = (None, 0, 0, 0)


def _refused(rc):
    msg = _lib.lib().ress_last_error()
    assert rc == -1 and b"2^32 threads or more" in msg, (rc, msg)


def test_cache_calls():
    """2^24 workgroups of 256 threads, from heads, pages or queries, are one too many."""
    L = _lib.lib()
    many = _CacheArgs(*[4096] * 12, 4, 4, 2, 1 << 23, 64, 1, 0)
    one = _CacheArgs(*[4096] * 12, 4, 4, 2, 1, 64, 1, 0)
    a, b = ctypes.addressof(many), ctypes.addressof(one)
    _refused(L.ress_kv_append(a, *F, *F, *Z, 2, 0, 1, None, None, 0, 1, None, None, None, None))
    _refused(L.ress_kv_append(b, *F, *F, *Z, 1, 0, 1 << 30, None, None, 0, 1, None, None, None, None))
    _refused(L.ress_kv_append(b, *F, *F, *F, 1, 1 << 26, 1, P, P, 4, 1, None, None, P, None))
    _refused(L.ress_kv_read(a, 2, 1, None, None, P, P, None))
    _refused(L.ress_kv_read(b, 1, 1 << 30, None, None, P, P, None))
    _refused(L.ress_kv_attend(a, *F, 2, 1 << 23, 1, None, None, 0, 0.125, 10, *F, None, 0, None))
    _refused(L.ress_kv_attend(a, *F, 2, 1 << 23, 40, None, None, 0, 0.125, 10, *F, None, 0, None))


@pytest.mark.parametrize("M,N", [(1 << 30, 64), (1 << 26, 1 << 20)])
def test_products(M, N):
    L = _lib.lib()
    size = L.ress_int8_linear_workspace_size(M, 64, N)
    assert size > 0
    _refused(L.ress_int8_linear(P, 64, 1, M, 64, N, P, P, None, 0, P, N, P, size, None))


@pytest.mark.gpu
def test_rows_of_several_launches(dev):
    """2^26 rows of 64 threads each are more than a launch holds: as the same rows in a short call."""
    import torch
    from ress_amd.int8 import quantize_tokens
    x = torch.randn(1024, 16, generator=torch.Generator().manual_seed(0)).to(dev, torch.bfloat16)
    codes, scale = quantize_tokens(x)
    many, scales = quantize_tokens(x.repeat((1 << 16) + 1, 1))
    assert (many.view(-1, 1024, 16) == codes).all() and (scales.view(-1, 1024) == scale).all()
