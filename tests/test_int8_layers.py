"""Int8Linear and quantize_linears as modules of a model (no GPU)."""

import pytest
import torch
import torch.nn as nn

from ress_amd import int8
from ress_amd.int8 import Int8Linear, quantize_linears


@pytest.mark.parametrize("cast", [nn.Module.half, nn.Module.bfloat16, nn.Module.float, nn.Module.double])
def test_weight_has_the_layers_present_type(cast):
    torch.manual_seed(0)
    layer = nn.Linear(32, 8).to(torch.bfloat16)
    q = Int8Linear(layer)
    assert q.weight.dtype == torch.bfloat16
    cast(layer)
    codes, scale, bias = q.codes.clone(), q.scale.clone(), q.bias.clone()
    assert cast(q) is q and q.weight.dtype == layer.weight.dtype
    assert torch.equal(q.codes, codes) and torch.equal(q.scale, scale) and torch.equal(q.bias, bias)
    assert q.scale.dtype == q.bias.dtype == torch.float32
    assert cast(nn.Sequential(q))[0].weight.dtype == layer.weight.dtype
    q.to("cpu")  # a move is no cast
    assert q.weight.dtype == layer.weight.dtype


class Shared(nn.Module):
    def __init__(self):
        super().__init__()
        self.a = nn.Linear(16, 16)
        self.b = self.a
        self.c = nn.Sequential(self.a, nn.Linear(16, 4))


def test_a_layer_under_several_names():
    """Replaced under each of them, by one layer; keep names it by any."""
    m = Shared()
    names = quantize_linears(m)
    assert sorted(names) == ["a", "b", "c.0", "c.1"]
    assert type(m.a) is Int8Linear and m.b is m.a and m.c[0] is m.a and m.c[1] is not m.a
    m = Shared()
    names = quantize_linears(m, keep=lambda name, linear: name == "b")
    assert sorted(names) == ["c.1"] and type(m.a) is nn.Linear and m.b is m.a and m.c[0] is m.a


def test_a_model_that_cannot_be_quantised_stays_whole():
    m = nn.Sequential(nn.Linear(16, 16), nn.Linear(16, 4), nn.Linear(16, 8))
    with torch.no_grad():
        m[1].weight[2, 3] = float("inf")
    with pytest.raises(ValueError, match="1: weight has values that are not finite"):
        quantize_linears(m)
    assert all(type(x) is nn.Linear for x in m)
    assert quantize_linears(m, keep=lambda name, linear: name == "1") == ["0", "2"]


def test_what_a_replaced_layer_keeps():
    """Its mode and its hooks."""
    m = nn.Sequential(nn.Linear(16, 16), nn.Linear(16, 4)).eval()
    calls = []
    m[0].register_forward_pre_hook(lambda mod, args: calls.append(type(mod)))
    m[0].register_forward_hook(lambda mod, args, out, **kw: calls.append(type(mod)))
    m[0].register_forward_pre_hook(lambda mod, args, kwargs: calls.append(kwargs), with_kwargs=True)
    quantize_linears(m)
    assert not m[0].training and not m[1].training
    m[0].forward = lambda x, act=None: x
    m[0](torch.zeros(2, 16), act="gelu")
    assert calls == [Int8Linear, {"act": "gelu"}, Int8Linear]


@pytest.mark.parametrize("to", [torch.bfloat16, torch.float16])
def test_autocast(monkeypatch, to):
    """As torch's own linear layer does: inputs of up to 32 bits are cast to autocast's type."""
    got = []
    monkeypatch.setattr(int8, "int8_linear", lambda x, *a: got.append(x))
    q = Int8Linear(nn.Linear(16, 4))
    x = torch.rand(3, 16)
    with torch.autocast("cpu", dtype=to):
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            q(x.to(dtype))
            assert got[-1].dtype == to and torch.equal(got[-1], x.to(dtype).to(to))
        q(x.double())
        assert got[-1].dtype == torch.float64
        with torch.autocast("cpu", enabled=False):
            q(x)
            assert got[-1] is x
    q(x)
    assert got[-1] is x


@pytest.mark.parametrize("which", ["scale", "bias"])
def test_weights_that_require_grad_are_refused(monkeypatch, which):
    """Like x that does: there is no backward pass, and the result would be cut off from them without a word."""
    calls = []
    monkeypatch.setattr(int8, "_rows", lambda x, name: x)
    monkeypatch.setattr(int8, "_workspace", lambda *a: 0)
    monkeypatch.setattr(int8._lib, "ptr", lambda t: t)
    monkeypatch.setattr(int8._lib, "call_on", lambda *a: calls.append(a))
    x, codes = torch.zeros(3, 16, dtype=torch.bfloat16), torch.zeros(4, 16, dtype=torch.int8)
    w = dict(scale=torch.ones(4), bias=torch.zeros(4))
    w[which].requires_grad_()
    with pytest.raises(RuntimeError, match=f"{which} requires grad"):
        int8.int8_linear(x, codes, w["scale"], w["bias"])
    assert not calls
    with torch.no_grad():
        int8.int8_linear(x, codes, w["scale"], w["bias"])
    int8.int8_linear(x, codes, w["scale"].detach(), w["bias"].detach())
    assert len(calls) == 2


def test_drift_matrices_of_8_bit_layers():
    """An attention whose projections are all 8-bit and whose norms have no weights has no parameters."""
    from ress_amd.aggregator import build_vggt_aggregator
    from ress_amd.projected import bake_and_attach_M
    model = build_vggt_aggregator(depth=2, dim=64, num_heads=1, device="cpu", dtype=torch.float32, wire=False)
    for block in model.aggregator.global_blocks:
        block.attn.q_norm = block.attn.k_norm = nn.Identity()
    quantize_linears(model.aggregator.global_blocks)
    M = bake_and_attach_M(model)
    for m, block in zip(M, model.aggregator.global_blocks):
        w = block.attn.proj.weight
        assert torch.equal(block.attn.M, m) and torch.equal(m[0], w.T @ w)


@pytest.mark.parametrize("way", ["weight_norm", "spectral_norm", "prune"])
def test_layers_whose_weight_a_hook_forms(monkeypatch, way):
    """The codes stand for the weight as it is; the hook that formed it has nothing to form any more."""
    from torch.nn.utils import prune
    monkeypatch.setattr(int8, "int8_linear", lambda x, codes, scale, bias, act: x @ (codes * scale[:, None]).t() + bias)
    torch.manual_seed(0)
    layer = nn.Linear(16, 4)
    if way == "prune":
        prune.l1_unstructured(layer, "weight", 0.5)
    else:
        getattr(nn.utils, way)(layer)
    layer.eval()
    x, seen = torch.rand(3, 16), []
    layer.register_forward_pre_hook(lambda mod, args: seen.append(1))
    m = nn.Sequential(layer)
    with torch.no_grad():
        want = m(x)
        assert quantize_linears(m) == ["0"]
        got = m(x)
    assert len(seen) == 2
    # half a step of 1/127 of the largest weight for each of 16 products, and fp32 sums
    assert ((got - want).abs() <= 16 * layer.weight.abs().max() / 254 + 1e-5).all()


class CountedGelu(nn.GELU):
    def forward(self, x):
        self.calls = getattr(self, "calls", 0) + 1
        return super().forward(x)


def test_mlp_leaves_no_activation_out(monkeypatch):
    """gelu is fused into the 8-bit layer where nothing else hangs on the activation module."""
    from ress_amd.aggregator import Mlp
    acts = []
    monkeypatch.setattr(int8, "int8_linear", lambda x, codes, scale, bias, act: (acts.append(act), x.new_zeros(*x.shape[:-1], len(codes)))[1])
    m = Mlp(16, 32)
    quantize_linears(m)
    x = torch.rand(3, 16)
    m(x)
    assert acts == ["gelu", None]
    for kind in ("register_forward_hook", "register_forward_pre_hook"):
        seen = []
        handle = getattr(m.act, kind)(lambda *a: seen.append(1) and None)
        m(x)
        assert seen == [1] and acts[-2:] == [None, None]
        handle.remove()
    m.act = CountedGelu()
    m(x)
    assert m.act.calls == 1 and acts[-2:] == [None, None]
