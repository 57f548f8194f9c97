"""The norm's backward entry refuses a workspace that is missing or not aligned before anything is launched (CPU; the addresses are never
used)."""

import pytest

from ress_amd import _lib, differentiable as df

P = 4096


def norm(rows=3):
    return df._NORM(P, 64, 0, 0, 0, 0, 0, 0, rows, 1, 1, 64, 1, 0, 0, 0, 0, 0, 0, P, P, 1e-5)


@pytest.mark.parametrize("at", [None, 4, P + 4, P + 8])
@pytest.mark.parametrize("which", [0, 1])
def test_a_workspace_that_cannot_be_used(at, which):
    L, g = _lib.lib(), df._STRIDED(P, 64, 0, 0)
    ends = [None, P, P][which:which + 2]
    rc = L.ress_layer_norm_bwd(norm(), g, None, P, None, None, *ends, at, 1 << 30, None)
    assert rc == -1 and b"workspace" in L.ress_last_error()
