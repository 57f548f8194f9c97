"""The paged cache's host side without a GPU: its layout's order, tables and refusals."""

import ctypes

import pytest
import torch

from kvcache_oracle import PAGE, v_token
from ress_amd import _lib
from ress_amd.kvcache import PagedKVCache, RotaryTable, _CacheArgs


def test_places_are_an_order():
    assert sorted(v_token(p) for p in range(PAGE)) == list(range(PAGE))
    # a lane (place // 16) holds, for each of the two products of 32 keys, four keys of each 16
    for p in range(PAGE):
        assert v_token(p) // 4 % 4 == p // 16 and v_token(p) // 32 == p // 8 % 2


def test_rotary_table():
    t = RotaryTable(64, 40, base=100.0, axes=2, device="cpu")
    assert tuple(t.table.shape) == (40, 2, 16)
    ang = 39 * 100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    assert (t.table[39, 0].double() - ang.cos()).abs().max() <= 2.0 ** -24
    assert (t.table[39, 1].double() - ang.sin()).abs().max() <= 2.0 ** -24
    assert tuple(RotaryTable(128, 3, axes=1, device="cpu").table.shape) == (3, 2, 64)
    for bad in (dict(head_dim=80, positions=4), dict(head_dim=64, positions=0), dict(head_dim=64, positions=4, axes=3),
                dict(head_dim=64, positions=4, base=1.0)):
        with pytest.raises(ValueError):
            RotaryTable(device="cpu", **bad)
    with pytest.raises(ValueError, match="table must"):
        RotaryTable.from_table(torch.zeros(4, 2, 32), 64, 2)


def test_a_cache_needs_the_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        PagedKVCache(4, 2, device="cpu")


def _args(**kw):
    a = _CacheArgs(*[4096] * 12, 4, 4, 2, 2, 64, 1, 0)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(head_dim=80), b"head_dim 80"), (dict(dtype=0), b"dtype code 0"), (dict(codes=2), b"codes 2"),
    (dict(n_pages=0), b"bad cache geometry"), (dict(max_pages=1 << 25), b"bad cache geometry"), (dict(tail_v=None), b"null buffer"), (dict(k_codes=4104), b"aligned"),
    (dict(max_seqs=1), b"more than the cache's 1 slots"),
])
def test_the_library_refuses_a_bad_cache(kw, msg):
    """Before any pointer is used: the addresses are never read."""
    L = _lib.lib()
    a = ctypes.addressof(x := _args(**kw))
    z = (None, 0, 0, 0)
    assert L.ress_kv_append(a, *z, *z, *z, 2, 0, 1, None, None, 0, 1, None, None, None, None) == -1
    assert msg in L.ress_last_error()
    assert L.ress_kv_read(a, 2, 1, None, None, None, None, None) == -1 and msg in L.ress_last_error()
    assert L.ress_kv_attend(a, *z, 2, 2, 1, None, None, 0, 0.125, 10, *z, None, 0, None) == -1
    assert msg in L.ress_last_error()
    del x


def test_the_library_refuses_bad_arguments():
    L = _lib.lib()
    x = _args()
    a, p, z = ctypes.addressof(x), ctypes.c_void_p(4096), (None, 0, 0, 0)
    f = (p, 0, 0, 64)
    for args, msg in (((*z, *f, *z, 2, 0, 1, None, None, 0, 1, None, None, None), b"null keys"),
                      ((*f, *f, *f, 2, 2, 1, None, None, 0, 1, None, None, p), b"without positions"),
                      ((*f, *f, *f, 2, 2, 1, p, p, 4, 1, None, None, None), b"go together"),
                      ((*f, *f, *z, 2, 0, 1, p, p, 4, 3, None, None, None), b"1 or 2 axes"),
                      ((*f, *f, *z, 2, 0, 1, p, None, 4, 1, None, None, None), b"at least one row"),
                      ((*f, *f, *z, 2, 0, -1, None, None, 0, 1, None, None, None), b"bad sizes")):
        assert L.ress_kv_append(a, *args, None) == -1 and msg in L.ress_last_error(), (msg, L.ress_last_error())
    assert L.ress_kv_attend(a, *f, 1, 3, 1, None, None, 0, 0.125, 10, *f, None, 0, None) == -1
    assert b"no multiple" in L.ress_last_error()
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert L.ress_kv_attend(a, *f, 1, 2, 1, None, None, 0, scale, 10, *f, None, 0, None) == -1
        assert b"scale" in L.ress_last_error()
    need = L.ress_kv_attend_workspace_size(a, 1, 2, 1, 100000)
    assert need > 0
    assert L.ress_kv_attend(a, *f, 1, 2, 1, None, None, 0, 0.125, 100000, *f, p, need - 1, None) == -1
    assert b"workspace needs" in L.ress_last_error()
    assert L.ress_kv_attend_workspace_size(a, 1, 3, 1, 100) == -1
    # nothing to do
    assert L.ress_kv_append(a, *z, *z, *z, 0, 0, 5, None, None, 0, 1, None, None, None, None) == 0
    assert L.ress_kv_attend(a, *z, 1, 2, 0, None, None, 0, 0.125, 10, *z, None, 0, None) == 0


def test_the_library_refuses_a_bad_linear():
    L = _lib.lib()
    p = ctypes.c_void_p(4096)
    ok = dict(x=p, dtype=1, M=20, K=64, N=8, w=p, ws=p, act=0, out=p, work=p, size=1 << 20)
    for kw, msg in ((dict(dtype=0), b"dtype code 0"), (dict(K=40), b"multiple of 16"), (dict(M=-1), b"multiple of 16"),
                    (dict(K=1 << 18), b"at most 131072"), (dict(N=-1), b"channel count"), (dict(act=2), b"act 2"),
                    (dict(x=None), b"null"), (dict(K=0), b"without elements"), (dict(w=ctypes.c_void_p(4104)), b"aligned"),
                    (dict(size=448 * 256), b"workspace needs"), (dict(work=None), b"workspace needs")):
        a = {**ok, **kw}
        assert L.ress_int8_linear(a["x"], 64, a["dtype"], a["M"], a["K"], a["N"], a["w"], a["ws"], None, a["act"], a["out"], 8,
                                  a["work"], a["size"], None) == -1
        assert msg in L.ress_last_error(), (kw, L.ress_last_error())
    assert L.ress_int8_linear_workspace_size(1, 64, 8) == 0
    assert L.ress_int8_linear_workspace_size(20, 64, 8) == (256 + 192) * 256 + 80
    assert L.ress_quantize_rows(p, 64, 1, 2, 64, p, 60, p, None) == -1 and b"8-byte aligned" in L.ress_last_error()


def test_stream_refusals():
    from ress_amd import FrameStream
    from ress_amd.aggregator import build_vggt_aggregator
    model = build_vggt_aggregator(depth=1, dim=64, num_heads=1, device="cpu", dtype=torch.float32)
    for bad in (dict(max_frames=0), dict(max_frames=2, batch=0)):
        with pytest.raises(ValueError, match="at least 1"):
            FrameStream(model, **bad)
    s = FrameStream(model, 2)
    for shape in ((2, 3, 28, 28), (1, 0, 3, 28, 28), (3, 28, 28)):
        with pytest.raises(ValueError, match="images must"):
            s.step(torch.zeros(shape))
    with pytest.raises(ValueError, match="do not fit"):
        s.step(torch.zeros(1, 3, 3, 28, 28))
    with pytest.raises(RuntimeError, match="no frame"):
        s.snapshot()
    with pytest.raises(ValueError, match="another stream"):
        s.restore((0, []))
    with pytest.raises(TypeError, match="dtype"):  # a cache of 32-bit keys
        s.step(torch.zeros(1, 3, 28, 28))


def test_special_tokens_of_later_frames():
    """Frame 0 has its own special tokens, every later one the shared ones, however the frames come."""
    from ress_amd.aggregator import build_vggt_aggregator
    agg = build_vggt_aggregator(depth=1, dim=64, num_heads=1, device="cpu", dtype=torch.float32).aggregator
    images = torch.rand(2, 3, 3, 28, 42)
    with torch.no_grad():
        whole, pos, grid = agg.tokens(images)
        assert grid == (2, 3) and tuple(whole.shape) == (2, 3, 11, 64) and tuple(pos.shape) == (11, 2)
        for i in range(3):
            x, p, _ = agg.tokens(images[:, i:i + 1], first_frame=i)
            assert torch.equal(x[:, 0], whole[:, i]) and torch.equal(p, pos)
