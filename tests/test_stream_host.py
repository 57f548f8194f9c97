"""FrameStream's steps without a GPU: a 32-bit model over plain caches in the place of the 8-bit ones."""

import pytest
import torch

from ress_amd import FrameStream, stream
from ress_amd.aggregator import build_vggt_aggregator
from ress_amd.wiring import wire_ress_attention


class PlainCache:
    """Keys and values as they come, rotated by the table; softmax over all of them."""

    def __init__(self, n_pages, heads, head_dim, **kw):
        self.k = self.v = None

    @staticmethod
    def _turn(x, pos, rope):
        out = []
        for a, part in enumerate(x.split(x.shape[-1] // rope.axes, -1)):
            cs = rope.table[pos[..., a]][:, None]
            x1, x2 = part.chunk(2, -1)
            out += [x1 * cs[..., 0, :] - x2 * cs[..., 1, :], x2 * cs[..., 0, :] + x1 * cs[..., 1, :]]
        return torch.cat(out, -1)

    def append(self, k, v, pos=None, rope=None, q=None):
        if rope is not None:
            k, q = self._turn(k, pos, rope), self._turn(q, pos, rope)
        self.k = k if self.k is None else torch.cat([self.k, k], 2)
        self.v = v if self.v is None else torch.cat([self.v, v], 2)
        return q

    def attend(self, q, out):
        out.copy_(torch.softmax(q @ self.k.transpose(2, 3) / q.shape[-1] ** 0.5, -1) @ self.v)

    def snapshot(self):
        return self.k, self.v

    def restore(self, snap):
        self.k, self.v = snap

    def release(self, slot):
        self.k = self.v = None


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(stream, "PagedKVCache", PlainCache)
    return build_vggt_aggregator(depth=3, dim=64, num_heads=1, device="cpu", dtype=torch.float32, wire=False)


def _frames(n, h=28, w=42):
    return torch.rand(1, n, 3, h, w, generator=torch.Generator().manual_seed(n))


def _dense(model, frames):
    with torch.no_grad():
        return model.aggregator(frames)


def test_all_frames_in_one_step(model):
    """fp32 sums in another order, of a few hundred terms of a residual stream of size one."""
    x = _frames(3)
    assert (FrameStream(model, 3).step(x) - _dense(model, x)).abs().max() <= 1e-4


@pytest.mark.parametrize("wired", [[1], [0, 2], [2, 1, 0], []])
def test_layers_wired_in_part(model, wired):
    """The stream runs every layer, in the model's order, whichever of them have been wired for the sparse path."""
    x = _frames(2)
    want = _dense(model, x)
    wire_ress_attention(model, [model.aggregator.global_blocks[i] for i in wired])
    assert (FrameStream(model, 2).step(x) - want).abs().max() <= 1e-4


def test_another_model_is_refused_when_the_stream_is_made(model):
    agg = model.aggregator
    for owner, name in ((model, "aggregator"), (agg, "frame_blocks"), (agg, "global_blocks"), (agg.global_blocks[1], "ls2"),
                        (agg.global_blocks[2], "norm1"), (agg.global_blocks[0].attn, "q_norm")):
        part = getattr(owner, name)
        delattr(owner, name)
        with pytest.raises(TypeError, match=name):
            FrameStream(model, 2)
        setattr(owner, name, part)
    last = agg.frame_blocks[2]
    del agg.frame_blocks[2]
    with pytest.raises(TypeError, match="2 frame blocks and 3 global"):
        FrameStream(model, 2)
    agg.frame_blocks.append(last)

    class Other(torch.nn.Module):  # an aggregator with blocks of its own and a forward over all frames at once
        def __init__(self):
            super().__init__()
            self.aggregator = torch.nn.Module()
            self.aggregator.frame_blocks, self.aggregator.global_blocks = agg.frame_blocks, agg.global_blocks

    with pytest.raises(TypeError, match="tokens"):
        FrameStream(Other(), 2)
    FrameStream(model, 2).step(_frames(2))


def test_no_frames_have_no_grid(model):
    """Taken back to no frame, a stream takes frames of another shape as a fresh one does (6 patches both)."""
    s = FrameStream(model, 3)
    s.step(_frames(1))
    s.reset()
    snap = s.snapshot()
    s.step(_frames(1))
    s.restore(snap)
    assert s.frames == 0
    x = _frames(2, 42, 28)
    assert (s.step(x) - _dense(model, x)).abs().max() <= 1e-4
    snap = s.snapshot()
    s.step(x[:, :1])
    s.restore(snap)
    with pytest.raises(ValueError, match="patch grid"):
        s.step(_frames(1))


@pytest.mark.parametrize("kind", ["register_forward_hook", "register_forward_pre_hook"])
@pytest.mark.parametrize("where", ["block", "attn"])
def test_hooks_that_would_not_run_are_refused(model, kind, where):
    """A step calls a global block's parts, so hooks on it or on its attention module would be left out."""
    s = FrameStream(model, 3)
    block = model.aggregator.global_blocks[1]
    handle = getattr(block if where == "block" else block.attn, kind)(lambda *a: None)
    with pytest.raises(RuntimeError, match="hooks"):
        s.step(_frames(1))
    assert s.frames == 0
    handle.remove()
    seen = []
    for m in (block.mlp, block.attn.proj, model.aggregator.frame_blocks[1]):  # these are called
        m.register_forward_hook(lambda *a: seen.append(1))
    s.step(_frames(1))
    assert len(seen) == 3 and s.frames == 1


def test_a_broken_step_is_no_snapshot(model):
    """After a step that ended in an error some layers hold its frame: nothing to come back to."""
    s = FrameStream(model, 4)
    s.step(_frames(1))
    good = s.snapshot()
    want = s.step(_frames(2))
    s.restore(good)
    mlp = model.aggregator.global_blocks[1].mlp
    handle = mlp.register_forward_pre_hook(lambda *a: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        s.step(_frames(2))
    handle.remove()
    with pytest.raises(RuntimeError, match="ended in an error"):
        s.snapshot()
    with pytest.raises(RuntimeError, match="ended in an error"):
        s.step(_frames(2))
    s.restore(good)
    assert torch.equal(s.step(_frames(2)), want)
    s.snapshot()


def test_a_capture_is_refused(monkeypatch, model):
    """Frames are counted on the host, when a call is made and not when a graph runs it."""
    s = FrameStream(model, 4)
    s.step(_frames(1))
    snap = s.snapshot()
    s.step(_frames(2))
    with monkeypatch.context() as m:
        m.setattr(stream, "_capturing", lambda: True, raising=False)
        for call in (lambda: s.step(_frames(1)), s.snapshot, lambda: s.restore(snap), s.reset):
            with pytest.raises(RuntimeError, match="not inside a graph capture"):
                call()
    assert s.frames == 3 and s.caches[0].k.shape[2] == 3 * 11
    s.restore(snap)
    assert s.frames == 1
