"""What kernels write as fp32 is fp32 whatever torch's default type is: a buffer of a 16-bit default would be half the
size that is written. Without a GPU: the buffers that reach the library calls."""

import os

import pytest
import torch

from ress_amd import int8, kvcache
from ress_amd.kvcache import PagedKVCache


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64])
def default(request):
    old = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(old)


def test_quantize_tokens(monkeypatch, default):
    got = []
    monkeypatch.setattr(int8, "_rows", lambda x, name: x)
    monkeypatch.setattr(int8._lib, "ptr", lambda t: t)
    monkeypatch.setattr(int8._lib, "call_on", lambda *a: got.append(a))
    codes, scale = int8.quantize_tokens(torch.zeros(3, 16, dtype=torch.bfloat16))
    assert scale.dtype == torch.float32 and codes.dtype == torch.int8
    assert got[0][-1].dtype == torch.float32


def test_cache(monkeypatch, default):
    """The constructor on the meta device, which allocates nothing."""
    real = torch.device

    class Torch:
        def __getattr__(self, name):
            return getattr(torch, name)

        @staticmethod
        def device(kind, index=None):  # the cache's own device: meta in its place
            return real("meta") if index is not None else real(kind)

    monkeypatch.setattr(kvcache, "torch", Torch())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(kvcache._lib, "ptr", lambda t: 4096)
    c = PagedKVCache(4, 2, max_seqs=3)
    assert c.device.type == "meta"
    for t in (c.k_scale, c.v_scale, c.tail_top):
        assert t.dtype == torch.float32
    assert c.tail_k.dtype == c.tail_v.dtype == torch.bfloat16
    for t in (c.table, c.held, c.lens, c._arrived, c._status):
        assert t.dtype == torch.int32


def _untyped(path):
    import ast
    made = ("empty", "zeros", "ones", "full", "empty_strided")
    return [f"{os.path.basename(path)}:{node.lineno}" for node in ast.walk(ast.parse(open(path).read()))
            if isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute) and node.func.attr in made
            and isinstance(node.func.value, ast.Name) and node.func.value.id == "torch"
            and not any(k.arg == "dtype" for k in node.keywords)]


def test_buffers_of_library_calls_name_their_type():
    """In every module that calls the library."""
    here = os.path.dirname(kvcache.__file__)
    paths = [os.path.join(here, f) for f in sorted(os.listdir(here)) if f.endswith(".py")]
    calling = [p for p in paths if "_lib.call" in open(p).read() or "_lib.ptr" in open(p).read()]
    assert len(calling) >= 7
    assert [x for p in calling for x in _untyped(p)] == []


def test_hyperparameter_check(default):
    from ress_amd.sparge import hyperparameter_check
    for x in (0.5, torch.rand(4)):
        assert hyperparameter_check(x, 4, "cpu").dtype == torch.float32
