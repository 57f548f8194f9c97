"""The kept index tables of a layer's blocks, used from several threads. CPU only."""

import torch

from ress_amd import training
from ress_amd.kernels import LayerGrid


def test_a_table_that_another_thread_clears(monkeypatch):
    """Between a thread's insertion and its return another one empties the tables."""

    class Emptied(dict):
        def __setitem__(self, key, value):
            super().__setitem__(key, value)
            self.clear()

    monkeypatch.setattr(training, "_plain_orders", Emptied())
    monkeypatch.setattr(training, "_capturing", lambda: False)
    monkeypatch.setattr(training._lib, "stream_handle", lambda device: 0)
    grid = LayerGrid(B=1, H=1, frames=2, P=20, S=5)
    got = training._layer_orders(grid, None, torch.device("cpu"))
    for a, b in zip(got[:4], training._orders(grid, None, torch.device("cpu"))[:4]):
        assert torch.equal(a, b)


def test_a_kept_table_is_the_same(monkeypatch):
    monkeypatch.setattr(training, "_plain_orders", {})
    monkeypatch.setattr(training, "_capturing", lambda: False)
    monkeypatch.setattr(training._lib, "stream_handle", lambda device: 0)
    grid = LayerGrid(B=1, H=1, frames=2, P=20, S=5)
    first = training._layer_orders(grid, None, torch.device("cpu"))
    assert training._layer_orders(grid, None, torch.device("cpu")) is first
    for frames in range(3, 20):
        training._layer_orders(LayerGrid(B=1, H=1, frames=frames, P=20, S=5), None, torch.device("cpu"))
        assert len(training._plain_orders) <= 8
