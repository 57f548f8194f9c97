"""The C entries of the operators with gradients, without a GPU: argument structs, workspaces, and what is refused is refused before
any pointer is used (the fake, aligned addresses below are never dereferenced)."""

import ctypes
import math
import struct

import pytest
import torch

import ress_amd as ress
from ress_amd import _lib, differentiable as df

P = 4096
OK = (P, 64, 64, 64)


class Strided(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("sb", ctypes.c_longlong), ("sh", ctypes.c_longlong), ("st", ctypes.c_longlong)]


class Attn(ctypes.Structure):
    _fields_ = ([(n, Strided) for n in ("q", "k", "v", "out")]
                + [(n, ctypes.c_int) for n in ("B", "q_heads", "kv_heads", "Tq", "Tk", "head_dim", "dtype", "causal")]
                + [("q_lens", ctypes.c_void_p), ("k_lens", ctypes.c_void_p), ("map", ctypes.c_void_p)]
                + [(n, ctypes.c_longlong) for n in ("sb", "sh", "sq", "sk")]
                + [("lse", ctypes.c_void_p), ("rest", ctypes.c_void_p), ("scale", ctypes.c_float)])


class Norm(ctypes.Structure):
    _fields_ = ([("x", Strided), ("branch", Strided)] + [(n, ctypes.c_int) for n in ("n0", "n1", "n2", "C", "dtype", "wide")]
                + [(n, ctypes.c_void_p) for n in ("gamma", "weight", "bias", "sum", "out", "mean", "rstd")] + [("eps", ctypes.c_float)])


class Rotary(ctypes.Structure):
    _fields_ = ([("x", Strided * 2), ("y", Strided * 2), ("heads", ctypes.c_int * 2)]
                + [(n, ctypes.c_int) for n in ("B", "n", "head_dim", "dtype", "axes", "rotary_dim", "interleaved", "inverse")]
                + [("pos", ctypes.c_void_p), ("sb", ctypes.c_longlong), ("st", ctypes.c_longlong), ("sa", ctypes.c_longlong),
                   ("table", ctypes.c_void_p), ("positions", ctypes.c_int), ("status", ctypes.c_void_p)])


@pytest.mark.parametrize("packed,c", [(df._STRIDED, Strided), (df._ATTN, Attn), (df._NORM, Norm), (df._ROTARY, Rotary)])
def test_packed_arguments_are_the_c_structs(packed, c):
    """Field by field: each of the struct's values is where the packed bytes have it."""
    leaves = []

    def walk(t, at):
        if hasattr(t, "_fields_"):
            for name, f in t._fields_:
                walk(f, at + getattr(t, name).offset)
        elif hasattr(t, "_length_"):
            for i in range(t._length_):
                walk(t._type_, at + i * ctypes.sizeof(t._type_))
        else:
            leaves.append((at, t))

    walk(c, 0)
    values = [1.5 + i if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(leaves)]
    raw = packed(*values)
    assert len(raw) == ctypes.sizeof(c)
    code = {ctypes.c_float: "f", ctypes.c_int: "i", ctypes.c_longlong: "q", ctypes.c_void_p: "q"}
    for (at, t), v in zip(leaves, values):
        assert struct.unpack_from("@" + code[t], raw, at)[0] == v


def attn(q=OK, k=OK, v=OK, out=OK, B=1, Hq=1, Hk=1, Tq=10, Tk=10, D=64, dtype=1, causal=0, ql=0, kl=0, m=(0, 0, 0, 0, 0), lse=0, rest=0, scale=0.125):
    return df._ATTN(*q, *k, *v, *out, B, Hq, Hk, Tq, Tk, D, dtype, causal, ql, kl, *m, lse, rest, scale)


def refused(rc, msg):
    got = _lib.lib().ress_last_error()
    assert rc == -1 and msg in got, (rc, got)


@pytest.mark.parametrize("kw,msg", [
    (dict(D=80), b"head_dim 80"), (dict(dtype=0), b"dtype code 0"), (dict(dtype=3), b"dtype code 3"), (dict(Hq=3, Hk=2), b"bad geometry"),
    (dict(Hk=0), b"bad geometry"), (dict(Tq=-1), b"bad geometry"), (dict(Tk=(1 << 26) + 1), b"2^26 tokens"),
    (dict(Tk=(1 << 20) + 1, m=(P, 0, 0, 0, 0)), b"under a map"), (dict(scale=0.0), b"scale"), (dict(scale=math.inf), b"scale"),
    (dict(scale=math.nan), b"scale"), (dict(q=(P + 8, 64, 64, 64)), b"aligned"), (dict(k=(P, 64, 64, 60)), b"aligned"),
    (dict(v=(P, 64, 64, 56)), b"apart"), (dict(out=(P, 64, 64, 1 << 24)), b"apart"), (dict(k=(0, 64, 64, 64)), b"aligned"),
    (dict(B=1 << 15, Hq=1 << 10, Hk=1 << 10), b"2^32 threads"), (dict(Hq=1 << 12, Tq=1 << 25), b"too many query heads"),
])
def test_attention_refusals(kw, msg):
    L, one = _lib.lib(), df._STRIDED(*OK)
    refused(L.ress_block_attn_fwd(attn(**kw), None, 0, None), msg)
    refused(L.ress_block_attn_bwd(attn(lse=P, rest=P, **kw), one, one, one, one, P, 1 << 62, None), msg)


def test_attention_refuses_without_arguments_workspace_or_statistics():
    L, one = _lib.lib(), df._STRIDED(*OK)
    refused(L.ress_block_attn_fwd(None, None, 0, None), b"null arguments")
    refused(L.ress_block_attn_bwd(attn(), None, one, one, one, None, 0, None), b"null arguments")
    refused(L.ress_block_attn_bwd(attn(), one, one, one, one, P, 1 << 20, None), b"rest and lse")
    refused(L.ress_block_attn_bwd(attn(lse=P, rest=P), one, one, one, one, None, 0, None), b"workspace")
    refused(L.ress_block_attn_bwd(attn(lse=P, rest=P), one, one, one, one, P + 4, 1 << 20, None), b"workspace")
    long = attn(Tk=20000)
    size = L.ress_block_attn_fwd_workspace_size(long)
    assert size > 0
    refused(L.ress_block_attn_fwd(long, P, size - 1, None), b"workspace")
    refused(L.ress_block_attn_fwd(long, None, size, None), b"workspace")


def test_attention_workspaces():
    L = _lib.lib()
    # tiles of 128 rows fill the card: nothing is cut. lse and delta of a row, the two maxima of a key/value head
    full = attn(B=4, Hq=64, Hk=64, Tq=1000, Tk=1000)
    assert L.ress_block_attn_fwd_workspace_size(full) == 0
    assert L.ress_block_attn_bwd_workspace_size(full) == 8 * 4 * 64 * 1000 + 8 * 4 * 64
    # one tile of 10 rows over 20,000 keys (313 steps of 64): 39 parts of 8 steps at least, 65 floats a row
    assert L.ress_block_attn_fwd_workspace_size(attn(Tk=20000)) == 39 * 10 * 65 * 4
    assert L.ress_block_attn_fwd_workspace_size(attn(D=80)) == -1 and L.ress_block_attn_bwd_workspace_size(attn(Hk=0)) == -1
    assert df._attn_workspace(False, attn(Tk=20000)[128:160], False) == 39 * 10 * 65 * 4
    mapped = attn(B=2, Hq=4, Hk=2, Tq=3000, Tk=5000, m=(P, 1, 1, 1, 1))
    assert df._attn_workspace(True, mapped[128:160], True) == L.ress_block_attn_bwd_workspace_size(mapped)


def norm(x=(P, 64, 0, 0), branch=(0, 0, 0, 0), n=(3, 1, 1), C=64, dtype=1, wide=0, p=(0, 0, 0, 0, P, 0, 0), eps=1e-5):
    return df._NORM(*x, *branch, *n, C, dtype, wide, *p, eps)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), b"dtype code 3"), (dict(C=0), b"rows of 0"), (dict(C=8193), b"rows of 8193"), (dict(n=(-1, 1, 1)), b"bad geometry"),
    (dict(n=(1, 0, 1)), b"bad geometry"), (dict(n=(1 << 20, 1 << 11, 1)), b"bad geometry"), (dict(n=(1, 1 << 16, 1 << 16)), b"bad geometry"),
    (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"), (dict(x=(0, 64, 0, 0)), b"null buffer"), (dict(p=(0,) * 7), b"null buffer"),
    (dict(branch=(P, 64, 0, 0)), b"null buffer"),
])
def test_norm_refusals(kw, msg):
    refused(_lib.lib().ress_layer_norm_fwd(norm(**kw), None), msg)


def test_norm_backward_refusals():
    L, g = _lib.lib(), df._STRIDED(P, 64, 0, 0)
    stats = (0, 0, 0, 0, 0, P, P)
    size = L.ress_layer_norm_bwd_workspace_size(norm())
    assert size == 3 * 64 * 4 * 3  # a part a row at most, of three sums
    assert df._norm_workspace(norm()[64:88]) == size
    assert L.ress_layer_norm_bwd_workspace_size(norm(n=(100000, 1, 1))) == 512 * 3 * 64 * 4
    refused(L.ress_layer_norm_bwd(norm(p=stats), g, None, P, None, None, P, None, P, size - 1, None), b"workspace")
    refused(L.ress_layer_norm_bwd(norm(), g, None, P, None, None, None, None, None, 0, None), b"null buffer")
    refused(L.ress_layer_norm_bwd(norm(p=stats), g, None, P, P, None, None, None, None, 0, None), b"no branch")
    refused(L.ress_layer_norm_bwd(None, g, None, P, None, None, None, None, None, 0, None), b"null arguments")


def rotary(x=OK, y=OK, x2=(0, 0, 0, 0), heads=(1, 0), B=1, n=1, D=64, dtype=1, axes=1, dims=64, pos=P, table=P, positions=4, status=P):
    return df._ROTARY(*x, *x2, *y, *x2, *heads, B, n, D, dtype, axes, dims, 0, 0, pos, 1, 1, 1, table, positions, status)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=0), b"dtype code 0"), (dict(D=65), b"head_dim 65"), (dict(D=258), b"head_dim 258"), (dict(axes=3), b"over 3 axes"),
    (dict(dims=66), b"66 dims"), (dict(dims=2, axes=2), b"2 dims"), (dict(dims=30, axes=2), b"30 dims"), (dict(positions=0), b"bad geometry"),
    (dict(heads=(1, 2)), b"null buffer"), (dict(pos=0), b"null buffer"), (dict(table=P + 4), b"unaligned table"), (dict(status=0), b"null buffer"),
    (dict(x=(0, 1, 1, 1)), b"null buffer"), (dict(B=1 << 15, n=1 << 16), b"2^32 threads"),
])
def test_rotary_refusals(kw, msg):
    refused(_lib.lib().ress_rotate(rotary(**kw), None), msg)


def test_operands_on_the_host_are_refused():
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    rope = ress.RotaryTable(64, 8, axes=1, device="cpu")
    for call in (lambda: ress.block_attention(x, x, x), lambda: ress.layer_norm(x), lambda: ress.add_layer_norm(x, x),
                 lambda: ress.rotate(x, torch.arange(4), rope)):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            call()


def test_nothing_to_do_is_done_without_a_launch():
    L = _lib.lib()
    assert L.ress_block_attn_fwd(attn(B=0), None, 0, None) == 0 and L.ress_block_attn_fwd(attn(Tq=0), None, 0, None) == 0
    assert L.ress_layer_norm_fwd(norm(n=(0, 1, 1)), None) == 0 and L.ress_rotate(rotary(n=0), None) == 0
