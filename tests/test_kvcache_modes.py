"""A cache made and used inside and outside torch.inference_mode()."""

import pytest
import torch

from ress_amd import kvcache
from ress_amd.kvcache import PagedKVCache


def test_buffers_are_no_inference_tensors(monkeypatch):
    """Those could not be changed outside of inference mode. The constructor on the meta device, which allocates nothing."""
    real = torch.device

    class Torch:
        def __getattr__(self, name):
            return getattr(torch, name)

        @staticmethod
        def device(kind, index=None):
            return real("meta") if index is not None else real(kind)

    monkeypatch.setattr(kvcache, "torch", Torch())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(kvcache._lib, "ptr", lambda t: 4096)
    with torch.inference_mode():
        c = PagedKVCache(4, 2, max_seqs=3)
    for t in (c.lens, c.held, c.table, c._state, c._status, c._arrived, c.k_codes, c.k_scale, c.tail_k, c.tail_top):
        assert not t.is_inference()


@pytest.mark.gpu
def test_calls_inside_and_outside(dev):
    x = torch.randn(1, 1, 200, 64, generator=torch.Generator().manual_seed(0)).to(dev, torch.bfloat16)

    def use(c, steps):
        out = []
        for mode in steps:
            with torch.inference_mode(mode):
                snap = c.snapshot()
                c.append(x, x)
                out.append(c.attend(x[:, :, :3]))
                c.restore(snap)
                c.append(x[:, :, :70], x[:, :, :70])
                out.append(c.attend(x[:, :, :3]))
                c.check()
        for mode in steps:
            with torch.inference_mode(mode):
                c.restore(snap)
                c.release(0)
                c.reserve(0, 100)
                c.append(x, x)
                snap = c.snapshot()
                out.append(c.attend(x[:, :, :3]))
        return out

    plain = use(PagedKVCache(16, 1, device=dev), (False, False, False))
    with torch.inference_mode():
        inside = PagedKVCache(16, 1, device=dev)
    for c, steps in ((inside, (False, True, False)), (PagedKVCache(16, 1, device=dev), (True, False, True))):
        for a, b in zip(plain, use(c, steps)):
            assert torch.equal(a, b)


def test_a_cache_made_inside_a_capture_is_refused(monkeypatch):
    """Its buffers would be cleared when the graph runs and not when it is made."""
    monkeypatch.setattr(kvcache, "_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(RuntimeError, match="not inside a graph capture"):
        PagedKVCache(4, 2)
