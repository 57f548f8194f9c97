"""Slots of a batch in every form that `slots` takes, and what the host knows of them afterwards (no GPU)."""

import numpy as np
import pytest
import torch

from host_cache import host_cache, tokens

FORMS = {
    "list": lambda ids: ids,
    "tuple": tuple,
    "tensor": torch.tensor,
    "array": np.array,
    "integers": lambda ids: [np.int64(i) for i in ids],
}


@pytest.mark.parametrize("form", FORMS)
def test_one_slot_after_a_batch_of_its_number(monkeypatch, form):
    """Slot 1 after a batch of one row (slot 0): another batch, whatever type its number has."""
    c = host_cache(monkeypatch)
    x = tokens(1, 10)
    c.append(x, x)
    c.append(x, x, slots=FORMS[form]([1]))
    assert c.held.tolist() == [1, 1]
    c.check()
    assert c.lens.tolist() == [10, 10]
    c._settle()
    assert c._bound == [10, 10]


@pytest.mark.parametrize("form", FORMS)
def test_several_slots_after_any_batch(monkeypatch, form):
    c = host_cache(monkeypatch, max_seqs=3)
    ids = FORMS[form]([2, 0])
    one, two = tokens(1, 10), tokens(2, 10)
    for slots in (None, [1, 2], c.slots([0, 1]), ids):
        c.append(two, two, slots=slots)
        c.append(two, two, slots=ids)
        c.append(one, one)
        c.append(two, two, slots=ids)
    c.check()
    want = c.lens.tolist()
    c._settle()
    assert c._bound == want == [80 + 40 + 30, 30, 80 + 20]  # twice ids each round, once slot 0, and the round's own


def test_the_same_batch_again_needs_no_new_bounds(monkeypatch):
    """The quick way of a batch that repeats: by its size where no slots are given, by its SlotBatch where they are."""
    c = host_cache(monkeypatch, max_seqs=3)
    x = tokens(2, 1)
    batch = c.slots([2, 1])
    for slots in (None, batch):
        c.append(x, x, slots=slots)
        for _ in range(5):
            c.append(x, x, slots=slots)
        assert c._lag == 5
    c._settle()
    assert c._bound == c.lens.tolist() == [6, 12, 6]
