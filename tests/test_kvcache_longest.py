"""ress_kv_attend's most_tokens past what the largest page table holds (no GPU): the keys are cut as for that."""

import ctypes

import pytest

from ress_amd import _lib
from ress_amd.kvcache import PAGE, _CacheArgs

LARGEST = PAGE * ((1 << 25) - 1)


@pytest.mark.parametrize("max_pages", [4, 5000])
@pytest.mark.parametrize("Hq,n", [(2, 1), (2, 5), (4, 100)])
def test_most_tokens(max_pages, Hq, n):
    L = _lib.lib()
    c = _CacheArgs(*[4096] * 12, max_pages, max_pages, 2, 2, 64, 1, 0)
    size = lambda most: L.ress_kv_attend_workspace_size(ctypes.addressof(c), 1, Hq, n, most)
    # parts of a positive number of pages: the workspace holds each part's outputs, maximum and sum
    parts, rest = divmod(size(LARGEST), 4 * Hq * n * (64 + 2))
    assert rest == 0 and 1 < parts <= 5 * 1024
    for most in range(LARGEST, 1 << 31, 9):
        assert size(most) == size(LARGEST), most
    assert size(0) == size(-5) == size(1) == 0
