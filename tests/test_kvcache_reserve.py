"""Pages taken and not taken: what a refused or failed call leaves behind (no GPU)."""

import pytest
import torch

from host_cache import host_cache, tokens
from ress_amd import kvcache


def test_reserve_refuses_a_capture(monkeypatch):
    """Its copy of page numbers cannot be recorded: refused before anything changes."""
    c = host_cache(monkeypatch)
    x = tokens(1, 10)
    c.append(x, x)
    before = (c.free_pages(), list(c._cap), c.table.clone(), c.held.clone())
    with monkeypatch.context() as m:
        m.setattr(kvcache, "_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="not inside a graph capture"):
            c.reserve(0, 200)
    assert before[:2] == (c.free_pages(), c._cap) and torch.equal(before[2], c.table) and torch.equal(before[3], c.held)
    c.append(tokens(1, 300), tokens(1, 300))
    c.check()
    assert c.lens.tolist() == [310, 0] and c.held.tolist() == [5, 0] and c.free_pages() == 3


@pytest.mark.parametrize("where", ["table", "held"])
def test_pages_are_taken_once_the_device_has_them(monkeypatch, where):
    """A copy that fails (no memory, say) leaves the pages free and the slot as it was."""
    c = host_cache(monkeypatch)
    x = tokens(1, 10)
    c.append(x, x)

    class Fails:
        def __init__(self, t):
            self.t = t

        def __getitem__(self, at):
            raise torch.OutOfMemoryError("no memory")

        __setitem__ = lambda self, at, value: self[at]

    real = getattr(c, where)
    setattr(c, where, Fails(real))
    with pytest.raises(torch.OutOfMemoryError):
        c.reserve(0, 200)
    with pytest.raises(torch.OutOfMemoryError):
        c.append(tokens(1, 100), tokens(1, 100))
    setattr(c, where, real)
    assert c.free_pages() == 7 and c._cap == [64, 0]
    c.append(tokens(1, 300), tokens(1, 300))
    c.check()
    assert c.lens.tolist() == [310, 0] and c.held.tolist() == [5, 0] and c.free_pages() == 3
    assert sorted(c.table[0, :5].tolist() + c._free) == list(range(8))


@pytest.mark.parametrize("n", [10, 100])
@pytest.mark.parametrize("again", [False, True])
def test_a_call_that_fails_appends_nothing(monkeypatch, n, again):
    """The library refuses or cannot launch: the host counts no token (a quick repeat of the last batch or not)."""
    fail = {}
    c = host_cache(monkeypatch, fail=fail)
    x, y = tokens(1, 10), tokens(1, n)
    c.append(x, x)
    fail["append"] = RuntimeError("ress_kv_append failed")
    for slots in (None, None if again else [1]):
        with pytest.raises(RuntimeError, match="failed"):
            c.append(y, y, slots=slots)
    fail.clear()
    if again:
        c.append(x, x)
    c._settle()
    assert c._bound == c.lens.tolist() == [20 if again else 10, 0]
    c.append(y, y)
    assert c._most == int(c.lens[0])
    c.check()


def _counts(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_padded_batches_that_fit_are_not_refused(monkeypatch):
    """Counts on the device, of which the host knows that they are at most n: where the pool has no pages for n of each,
    what counts is what they are."""
    c = host_cache(monkeypatch, n_pages=3)
    x = tokens(2, 100)
    c.append(x, x, new_lens=_counts(100, 20))
    c.check()
    assert c.lens.tolist() == [100, 20] and c.free_pages() == 0
    c.append(x, x, new_lens=_counts(28, 44))  # to the last place
    c.check()
    assert c.lens.tolist() == [128, 64]
    with pytest.raises(RuntimeError, match="0 free pages of 3, 1 are needed"):
        c.append(x, x, new_lens=_counts(0, 1))
    assert c.lens.tolist() == [128, 64]
    c.append(x, x, new_lens=_counts(0, -3))  # taken as none
    c.check()
    c = host_cache(monkeypatch, n_pages=8, max_pages=2)  # past max_len: dropped and reported, as documented
    c.append(x, x, new_lens=_counts(100, 20))
    c.append(x, x, new_lens=_counts(100, 20))
    assert c.lens.tolist() == [128, 40]
    with pytest.raises(RuntimeError, match="dropped"):
        c.check()


def test_a_capture_after_padded_batches(monkeypatch):
    """The host's estimates count the padding; inside a capture, where lengths cannot be read, they refuse nothing that the
    reserved pages may hold. What does not fit is dropped and reported when the graph runs."""
    c = host_cache(monkeypatch)
    x = tokens(1, 50)
    c.reserve(0, 128)
    for _ in range(4):
        c.append(x, x, new_lens=_counts(5))
    assert c.lens.tolist() == [20, 0]
    with monkeypatch.context() as m:
        m.setattr(kvcache, "_capturing", lambda: True)
        c.append(x, x)
        with pytest.raises(RuntimeError, match="reserved before"):
            c.append(tokens(1, 129), tokens(1, 129))  # never fits
        with pytest.raises(RuntimeError, match="reserved before"):
            c.append(tokens(2, 1), tokens(2, 1))  # slot 1 has no pages
    assert c.lens.tolist() == [70, 0]
    c.append(x, x)
    c.check()
    assert c.lens.tolist() == [120, 0]
    # where the lengths are known, a capture that cannot run once is refused
    d = host_cache(monkeypatch)
    d.append(x, x)
    with monkeypatch.context() as m:
        m.setattr(kvcache, "_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="reserved before"):
            d.append(x, x)
