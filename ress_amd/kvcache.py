"""A paged 8-bit key/value cache and the attention over it, for sequences that arrive in pieces.

The block-sparse layers attend over every frame of a scene at once. A scene that arrives frame by
frame (or a decoder that makes one token at a time) keeps the keys and values of what it has seen
and lets the new tokens attend to them:

    cache = PagedKVCache(n_pages=400, n_kv_heads=16, max_seqs=1, max_len=25_600)
    rope = RotaryTable(64, 64, base=100.0, axes=2)
    q = cache.append(k, v, pos=pos, rope=rope, q=q)   # rotates q and k, stores k and v
    out = cache.attend(q)                             # (B, Hq, n, D)

A page is 64 tokens (the framework's key block) of one key/value head, in 8 bits (int8, or e4m3 with
codes="fp8") with one scale for its keys and one for its values: half the memory of 16-bit keys and
values, and half the bytes that attention reads. The tokens of a sequence's unfinished page stay in
16 bits and are quantised once, when the page is full, so the cache's contents depend on the tokens
alone and not on how they were split over calls.

Every method works on torch's current stream of the cache's device. These wait for the device: lengths and
check; reserve, and an append that needs pages (a small copy of page numbers; once the host no longer knows the
lengths, as with counts on the device, it reads them first; after a captured append each eager one does); and
every argument that comes from the host (slots or new_lens as a list, pos on the CPU), whose copy waits: a
decoding loop passes a SlotBatch and tensors on the device. Calls that change a cache (append, reserve, restore,
release) must be ordered one after the other, as on one stream, and so must two captured graphs that append to
one cache; attend and read only read it, and must be ordered with the calls that change the slots they read.

The reference has no counterpart: it attends over all frames at once.
"""

import ctypes
import math
import weakref

import torch

from ress_amd import _lib

PAGE = 64
MOST_ROWS = 1 << 30  # of an operand, over batch and heads
CODES = {"int8": 0, "fp8": 1}
DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_STATUS = (
    (1, "tokens were dropped: their sequence has no page reserved for them (reserve)"),
    (2, "a position lies outside the rotation table (it was clamped into it)"),
    (4, "a page number lies outside the pool (the table was changed from outside)"),
    (8, "a page holds a key or value that is not finite (queries that see it get NaN)"),
    (16, "a slot lies outside the cache (a SlotBatch's tensor was changed, or freed under a recorded graph)"),
)


def _capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


class _CacheArgs(ctypes.Structure):
    """ress_kv_cache of include/ress_hip.h."""

    _fields_ = [(name, ctypes.c_void_p) for name in (
        "k_codes", "v_codes", "k_scale", "v_scale", "tail_k", "tail_v", "tail_top", "table", "held", "lens", "arrived",
        "status")] + [(name, ctypes.c_int) for name in (
            "n_pages", "max_pages", "max_seqs", "kv_heads", "head_dim", "dtype", "codes")]


class RotaryTable:
    """Cosines and sines of positions 0..positions-1, formed in 64 bits and rounded once, for
    PagedKVCache.append. axes=1: the rotary embedding of a token's index over the whole head dim;
    axes=2: of a row and a column over its two halves (this package's RoPE2D). Dims i and i + d/2 of
    an axis of d dims turn together by position * base^(-2i/d)."""

    def __init__(self, head_dim, positions, base=100.0, axes=2, device="cuda"):
        d = self._check(head_dim, axes)
        if int(positions) < 1 or not float(base) > 1.0:
            raise ValueError(f"a rotation table needs at least one position and a base above 1, got {positions} and {base}")
        inv = float(base) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        ang = torch.arange(int(positions), dtype=torch.float64)[:, None] * inv
        self.table = torch.stack([ang.cos(), ang.sin()], 1).float().to(device)
        self.head_dim, self.axes = head_dim, axes

    @staticmethod
    def _check(head_dim, axes):
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if axes not in (1, 2):
            raise ValueError(f"axes must be 1 or 2, got {axes}")
        return head_dim // axes

    @classmethod
    def from_table(cls, table, head_dim, axes):
        """From (positions, 2, head_dim / 2 / axes) fp32 cosines and sines on the device."""
        d = cls._check(head_dim, axes)
        if table.dtype != torch.float32 or table.dim() != 3 or tuple(table.shape[1:]) != (2, d // 2) or not len(table):
            raise ValueError(f"table must be (positions, 2, {d // 2}) float32, got {tuple(table.shape)} {table.dtype}")
        self = cls.__new__(cls)
        self.table, self.head_dim, self.axes = table.contiguous(), head_dim, axes
        return self


class SlotBatch:
    """The slots that the rows of a batch belong to (PagedKVCache.slots)."""

    def __init__(self, ids, device):
        self.ids = ids
        self.tensor = torch.tensor(ids, dtype=torch.int32, device=device)

    def __len__(self):
        return len(self.ids)


class Snapshot:
    """What PagedKVCache.restore needs to take appended tokens back."""

    def __init__(self, state, bounds, guessed, serial):
        self.state, self.bounds, self.guessed, self.serial = state, bounds, guessed, serial
        self.alive = True


class PagedKVCache:
    """`max_seqs` sequences (slots) of at most `max_len` tokens each (rounded up to whole pages; default: the
    whole pool) in a pool of `n_pages` pages of 64 tokens. dtype: bfloat16 or float16, the type of the keys, values and
    queries; codes: "int8" or "fp8" (e4m3). head_dim: 64 or 128."""

    def __init__(self, n_pages, n_kv_heads, head_dim=64, max_seqs=1, max_len=None, dtype=torch.bfloat16,
                 codes="int8", device="cuda"):
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if dtype not in DTYPES:
            raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
        if codes not in CODES:
            raise ValueError(f"codes must be one of {tuple(CODES)}, got {codes!r}")
        for name, x in (("n_pages", n_pages), ("n_kv_heads", n_kv_heads), ("max_seqs", max_seqs)):
            if int(x) < 1:
                raise ValueError(f"{name} must be at least 1, got {x}")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("a PagedKVCache lives on the GPU")
        if _capturing():
            raise RuntimeError("a cache is cleared when it is made: not inside a graph capture")
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        self.n_pages, self.kv_heads, self.head_dim, self.max_seqs = int(n_pages), int(n_kv_heads), head_dim, int(max_seqs)
        self.max_pages = self.n_pages if max_len is None else min(self.n_pages, -(-int(max_len) // PAGE))
        if not 1 <= self.max_pages < 1 << 25:
            raise ValueError(f"max_len must be 1 to {(PAGE << 25) - PAGE} tokens, got {max_len}")
        self.dtype, self.codes = dtype, codes
        P, H, D, S, dev = self.n_pages, self.kv_heads, head_dim, self.max_seqs, self.device
        code_t = torch.int8 if codes == "int8" else torch.float8_e4m3fn
        with torch.inference_mode(False):  # buffers that calls outside of inference mode may change too
            self.k_codes = torch.zeros(P, H, PAGE, D, dtype=torch.int8, device=dev).view(code_t)
            self.v_codes = torch.zeros(P, H, D, PAGE, dtype=torch.int8, device=dev).view(code_t)
            self.k_scale = torch.zeros(P, H, dtype=torch.float32, device=dev)
            self.v_scale = torch.zeros(P, H, dtype=torch.float32, device=dev)
            # what an append overwrites lies in one buffer, so that a snapshot is one copy
            tail = S * H * PAGE * D * 2
            self._state = torch.zeros(2 * tail + 4 * S * H + 4 * S, dtype=torch.uint8, device=dev)
            self.tail_k = self._state[:tail].view(dtype).view(S, H, PAGE, D)
            self.tail_v = self._state[tail:2 * tail].view(dtype).view(S, H, D, PAGE)
            self.tail_top = self._state[2 * tail:2 * tail + 4 * S * H].view(torch.float32).view(S, H)
            self.lens = self._state[2 * tail + 4 * S * H:].view(torch.int32)
            self.table = torch.full((S, self.max_pages), -1, dtype=torch.int32, device=dev)
            self.held = torch.zeros(S, dtype=torch.int32, device=dev)
            self._arrived = torch.zeros(S, 32, dtype=torch.int32, device=dev)
            self._status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._free = list(range(P - 1, -1, -1))
        self._pages = [[] for _ in range(S)]
        self._bound = [0] * S     # no slot holds more tokens than this
        self._cap = [0] * S       # tokens that a slot's pages have room for
        # Appends of one batch that needed no pages, not yet in _bound: `_lag` tokens for each slot of `_key` (a
        # SlotBatch, or B for slots 0..B-1), which has room for `_slack` more and holds at most `_most`.
        self._key, self._lag, self._slack, self._most = None, 0, 0, 0
        self._captured = False    # captured work moves lengths that the host does not see
        self._guessed = False     # _bound counts padding (counts on the device)
        self._snapshots = weakref.WeakSet()
        self._serial = 0
        p = _lib.ptr
        self._args = _CacheArgs(p(self.k_codes), p(self.v_codes), p(self.k_scale), p(self.v_scale), p(self.tail_k),
                                p(self.tail_v), p(self.tail_top), p(self.table), p(self.held), p(self.lens),
                                p(self._arrived), p(self._status), P, self.max_pages, S, H, D, DTYPES[dtype],
                                CODES[codes])
        self._handle = ctypes.addressof(self._args)

    # ---- slots and pages ----------------------------------------------------
    def slots(self, ids):
        """The slots of a batch's rows, checked (in range, none twice) and on the device: make it once
        for calls that repeat."""
        ids = [int(i) for i in ids]
        self._not_capturing("slots", "a SlotBatch (slots)")
        if any(not 0 <= i < self.max_seqs for i in ids):
            raise IndexError(f"slots must lie in 0..{self.max_seqs - 1}, got {ids}")
        if len(set(ids)) != len(ids):
            raise ValueError(f"a slot may appear once in a batch, got {ids}")
        return SlotBatch(ids, self.device)

    def _batch(self, slots, B):
        """(slots on the host, on the device or None, the batch's key: B where no slots are given, else a SlotBatch)."""
        if slots is None:
            if B > self.max_seqs:
                raise ValueError(f"a batch of {B} needs {B} slots, the cache has {self.max_seqs}")
            return range(B), None, B
        if not isinstance(slots, SlotBatch):
            slots = self.slots(slots)
        if len(slots) != B or slots.tensor.device != self.device or any(i >= self.max_seqs for i in slots.ids):
            raise ValueError(f"the batch has {B} rows and {len(slots)} slots, or they belong to another cache")
        return slots.ids, slots.tensor, slots

    @staticmethod
    def _not_capturing(name, want):
        if _capturing():
            raise RuntimeError(f"inside a graph capture {name} must be {want} made before it")

    def _settle(self):
        """Brings _bound up to date."""
        if self._lag:
            for i in range(self._key) if isinstance(self._key, int) else self._key.ids:
                self._bound[i] = min(self._bound[i] + self._lag, self._cap[i])
        self._key, self._lag = None, 0

    def free_pages(self):
        return len(self._free)

    def lengths(self):
        """Tokens in each slot (waits for the device)."""
        got = self.lens.tolist()
        self._key, self._lag = None, 0
        self._bound[:] = got
        self._guessed = False
        return got

    def _room(self, ids, more, counts=None):
        """Pages for more[i] further tokens in each slot. Bounds that the host only estimates (padded
        batches, captured appends) are read from the device before pages are taken for them or anything is
        refused. counts: `more` is itself an estimate of these counts on the device; a slot is then given no more than
        max_len, and they are read where the pool has too little for the estimate."""
        most = PAGE * self.max_pages

        def wanted():
            need = {i: self._bound[i] + m for i, m in zip(ids, more)}
            return need if counts is None else {i: min(n, most) for i, n in need.items()}

        capturing, known = _capturing(), not (self._captured or self._guessed)
        if not known and not capturing:
            self.lengths()
        # lengths that cannot be read inside a capture refuse nothing that the slot's pages may hold
        need = wanted() if known or not capturing else dict(zip(ids, more))
        if all(n <= self._cap[i] for i, n in need.items()):
            return
        if capturing:
            raise RuntimeError("an append inside a graph capture needs its pages reserved before (reserve)")
        if not self._fits(need):
            self.lengths()
            if counts is not None and not self._fits(wanted()):
                more = [min(max(c, 0), m) for c, m in zip(counts.tolist(), more)]
            need = wanted()
            self._fits(need, refuse=True)
        for i, n in need.items():
            self._take(i, n)

    def _fits(self, need, refuse=False):
        """Whether every slot of {slot: tokens} can have its pages, all together."""
        over = [i for i, n in need.items() if n > PAGE * self.max_pages]
        if over:
            if refuse:
                raise ValueError(f"slot {over[0]} cannot hold {need[over[0]]} tokens: max_len is {PAGE * self.max_pages}")
            return False
        new = sum(max(0, -(-n // PAGE) - len(self._pages[i])) for i, n in need.items())
        if new > len(self._free):
            if refuse:
                raise RuntimeError(f"the cache has {len(self._free)} free pages of {self.n_pages}, {new} are needed")
            return False
        return True

    def _take(self, slot, n_tokens):
        have, need = len(self._pages[slot]), -(-n_tokens // PAGE)
        if need <= have:
            return
        new = self._free[have - need:][::-1]
        with torch.cuda.device(self.device):
            self.table[slot, have:need] = torch.tensor(new, dtype=torch.int32, device=self.device)
            self.held[slot:slot + 1].fill_(need)
        # the device has them: a copy that failed leaves them free
        del self._free[have - need:]
        self._pages[slot] += new
        self._cap[slot] = PAGE * need

    def reserve(self, slot, n_tokens):
        """Pages for n_tokens tokens of a slot in all (those it holds included). append reserves by
        itself what it needs, except inside a graph capture."""
        if not 0 <= slot < self.max_seqs:
            raise IndexError(f"slot must lie in 0..{self.max_seqs - 1}, got {slot}")
        if _capturing():
            raise RuntimeError("reserve copies page numbers from the host: not inside a graph capture")
        self._settle()
        self._fits({slot: int(n_tokens)}, refuse=True)
        self._take(slot, int(n_tokens))

    def release(self, slot):
        """Empties a slot and gives its pages back. Work that reads them has to be ordered before."""
        if not 0 <= slot < self.max_seqs:
            raise IndexError(f"slot must lie in 0..{self.max_seqs - 1}, got {slot}")
        if _capturing():
            raise RuntimeError("release gives pages back at once: not inside a graph capture")
        self._settle()
        with torch.cuda.device(self.device):
            self.held[slot:slot + 1].fill_(0)
            self.lens[slot:slot + 1].fill_(0)
            self.table[slot].fill_(-1)
        self._free += reversed(self._pages[slot])
        self._pages[slot] = []
        self._bound[slot] = self._cap[slot] = 0
        for snap in self._snapshots:
            snap.alive = False

    def snapshot(self):
        """The state that restore goes back to (a copy of the unfinished pages and the lengths). Recorded in a graph, it is
        that of the graph's last run."""
        self._settle()
        self._serial += 1
        self._captured = self._captured or _capturing()
        snap = Snapshot(self._state.clone(), list(self._bound), self._guessed, self._serial)
        self._snapshots.add(snap)
        return snap

    def restore(self, snapshot):
        """Takes back every token appended since the snapshot, in every slot; pages stay reserved. A
        snapshot holds until a slot is released or an older one is restored."""
        if snapshot not in self._snapshots:
            raise ValueError("the snapshot belongs to another cache")
        if not snapshot.alive:
            raise RuntimeError("the snapshot no longer holds: a slot was released, or an older snapshot restored, since")
        self._captured = self._captured or _capturing()
        self._state.copy_(snapshot.state)
        self._key, self._lag = None, 0
        self._bound[:], self._guessed = snapshot.bounds, snapshot.guessed
        if snapshot.serial < self._serial:
            for snap in self._snapshots:
                if snap.serial > snapshot.serial:
                    snap.alive = False

    def check(self):
        """Raises if a call since the last check met something it could not do (waits for the device)."""
        word = int(self._status.item())
        if word:
            self._status.zero_()
            raise RuntimeError("PagedKVCache: " + "; ".join(text for bit, text in _STATUS if word & bit))

    # ---- operands -----------------------------------------------------------
    def _operand(self, t, name, heads=None, like=None):
        """Strides of a (B, heads, n, head_dim) operand; raises what is wrong with one."""
        if torch.is_tensor(t) and t.dtype is self.dtype and t.device == self.device and t.dim() == 4:
            B, H, n, D = t.shape
            st = t.stride()
            if (D == self.head_dim and st[3] == 1 and (heads is None or H == heads)
                    and (like is None or (B == like.shape[0] and n == like.shape[2])) and B * H * n <= MOST_ROWS
                    and not (t.requires_grad and torch.is_grad_enabled())):
                return st[:3]
        if not torch.is_tensor(t) or not t.is_cuda:
            raise RuntimeError(f"{name} must be a device tensor (the cache lives on the GPU)")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.dtype != self.dtype:
            raise TypeError(f"{name} must be {self.dtype} like the cache, got {t.dtype}")
        if t.dim() != 4 or t.shape[3] != self.head_dim or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{name} must be (B, {heads or 'heads'}, n, {self.head_dim}), got {tuple(t.shape)}")
        if like is not None and (t.shape[0], t.shape[2]) != (like.shape[0], like.shape[2]):
            raise ValueError(f"{name} must have the batch and tokens of k, ({like.shape[0]}, {like.shape[2]}), got {tuple(t.shape)}")
        if t.shape[0] * t.shape[1] * t.shape[2] > MOST_ROWS:
            raise ValueError(f"{name} must have at most {MOST_ROWS} rows, got {tuple(t.shape)}")
        if t.stride(3) != 1:
            raise ValueError(f"{name} must have a unit-stride head dim")
        raise RuntimeError(f"{name} requires grad: the cache has no backward pass (use torch.no_grad())")

    def _new_lens(self, new_lens, B, n):
        """(device int32 (B,) or None, counts on the host: empty where they are n or not known but for that)."""
        if new_lens is None:
            return None, ()
        if torch.is_tensor(new_lens):
            if new_lens.device != self.device or new_lens.dtype != torch.int32 or tuple(new_lens.shape) != (B,):
                raise ValueError(f"new_lens must be ({B},) int32 on {self.device}, got {tuple(new_lens.shape)} "
                                 f"{new_lens.dtype} on {new_lens.device}")
            return new_lens.contiguous(), ()
        self._not_capturing("new_lens", "an int32 tensor")
        got = [int(x) for x in new_lens]
        if len(got) != B or any(not 0 <= x <= n for x in got):
            raise ValueError(f"new_lens must be {B} counts of 0..{n}, got {got}")
        return torch.tensor(got, dtype=torch.int32, device=self.device), got

    def _call(self, name, *args):
        _lib.call_on(self.device, name, *args)

    # ---- the operators ------------------------------------------------------
    def append(self, k, v, pos=None, rope=None, q=None, slots=None, new_lens=None):
        """Appends n tokens to each sequence: k, v (B, kv_heads, n, head_dim), any strides with unit-stride
        dims. Row b goes to slots[b] (default: slot b); new_lens, (B,) int32 on the device or a list: row
        b has that many tokens, the others of its n are padding. Pages are reserved as needed; a call that
        does not fit is refused whole. With counts on the device, which the host does not see, tokens past
        max_len are dropped instead and reported by check().

        pos (B, n) or (B, n, axes) with a RotaryTable `rope`: k, and the queries q (B, heads, n, head_dim) if
        given, are rotated by it on the way. Returns the rotated queries (zeros in padding), or None.
        Positions outside the table are clamped and reported by check()."""
        ks = self._operand(k, "k", self.kv_heads)
        vs = self._operand(v, "v", self.kv_heads, like=k)
        B, n = k.shape[0], k.shape[2]
        ids, slot_t, key = self._batch(slots, B)
        if (pos is None) != (rope is None):
            raise ValueError("pos and rope go together")
        qs, q_out, q_heads = (0, 0, 0), None, 0
        if q is not None:
            if pos is None:
                raise ValueError("queries are rotated beside the keys: q needs pos and rope")
            qs = self._operand(q, "q", like=k)
            q_heads = q.shape[1]
        axes, positions, table = 1, 0, None
        if pos is not None:
            axes, table = rope.axes, rope.table
            positions = table.shape[0]
            if rope.head_dim != self.head_dim or table.device != self.device:
                raise ValueError(f"rope is for head_dim {rope.head_dim} on {table.device}, the cache has {self.head_dim} on {self.device}")
            want = ((B, n), (B, n, 1)) if axes == 1 else ((B, n, 2),)
            if pos.shape not in want or pos.is_floating_point():
                raise ValueError(f"pos must be {want[0]} whole numbers, got {tuple(pos.shape)} {pos.dtype}")
            if pos.device != self.device:
                self._not_capturing("pos", "a tensor on the cache's device")
            if pos.dtype is not torch.int64 or pos.device != self.device:
                pos = pos.to(device=self.device, dtype=torch.int64)
            pos = pos.contiguous()
        lens_t, counts = self._new_lens(new_lens, B, n)
        if q is not None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        if B == 0 or n == 0:
            return q_out
        guess = lens_t is not None and not counts
        capturing = _capturing()
        same = not counts and key == self._key and n <= self._slack and not self._captured and not capturing
        bound, cap = self._bound, self._cap
        if not same:
            self._settle()
            counts = counts or [n] * B
            if self._captured or capturing or any(bound[i] + c > cap[i] for i, c in zip(ids, counts)):
                self._room(ids, counts, lens_t if guess else None)
            self._captured = self._captured or capturing
        P = _lib.ptr
        self._call("ress_kv_append", self._handle, P(k), *ks, P(v), *vs, P(q), *qs, B, q_heads, n, P(pos), P(table),
                   positions, axes, P(slot_t), P(lens_t), P(q_out))
        # counted once the call is under way: one that fails appends nothing
        if same:
            self._lag += n
            self._slack -= n
            self._most += n
        elif not capturing:
            for i, c in zip(ids, counts):
                bound[i] = min(bound[i] + c, cap[i])
            self._key, self._slack = key, min(cap[i] - bound[i] for i in ids)
            self._most = max(bound[i] for i in ids)
        self._guessed = self._guessed or guess
        return q_out

    def read(self, n, slots=None, start=None, batch=None):
        """(k, v), each (B, kv_heads, n, head_dim): the last n tokens of each sequence as the cache holds
        them, or those from start[b] on ((B,) int32 on the device). Zeros where a sequence has no token.
        B: the slots given, else the entries of start, else `batch` (default: every slot)."""
        if slots is not None and not isinstance(slots, SlotBatch):
            slots = self.slots(slots)
        B = len(slots) if slots is not None else len(start) if start is not None else self.max_seqs if batch is None else batch
        _, slot_t, _ = self._batch(slots, B)
        n = int(n)
        if n < 0:
            raise ValueError(f"n must not be negative, got {n}")
        if start is not None and (not torch.is_tensor(start) or start.device != self.device or start.dtype != torch.int32
                                  or tuple(start.shape) != (B,)):
            raise ValueError(f"start must be ({B},) int32 on {self.device}")
        start = None if start is None else start.contiguous()
        k = torch.empty(B, self.kv_heads, n, self.head_dim, dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        if k.numel():
            self._call("ress_kv_read", self._handle, B, n, _lib.ptr(slot_t), _lib.ptr(start), _lib.ptr(k), _lib.ptr(v))
        return k, v

    def attend(self, q, slots=None, causal=False, new_lens=None, scale=None, out=None):
        """softmax(scale q K^T) V of the queries q (B, heads, n, head_dim; heads a multiple of kv_heads, query
        head h reading key/value head h / (heads / kv_heads)) over what the cache holds. The queries belong
        to the last n tokens of their sequence (the last new_lens[b] of them, the other rows being padding);
        they see all of it, or with causal=True the tokens up to their own. scale: 1/sqrt(head_dim). The softmax's weights
        (and float16 values, scaled) are rounded to the cache's type before they meet; maxima and sums are fp32.

        Returns (B, heads, n, head_dim), zeros in padding and in rows that see nothing; a given `out` is
        written in place, its padding left as it was; it shares no memory with q."""
        qs = self._operand(q, "q")
        B, Hq, n, D = q.shape
        if Hq == 0 or Hq % self.kv_heads:
            raise ValueError(f"q must have a multiple of {self.kv_heads} heads, got {Hq}")
        ids, slot_t, key = self._batch(slots, B)
        lens_t, _ = self._new_lens(new_lens, B, n)
        scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
        if not 0.0 < scale < math.inf:
            raise ValueError(f"scale must be positive and finite, got {scale}")
        if out is None:
            out = (torch.empty if lens_t is None else torch.zeros)(q.shape, dtype=q.dtype, device=self.device)
            os = out.stride()[:3]
        else:
            os = self._operand(out, "out")
            if out.shape != q.shape:
                raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
            if any(s == 0 and m > 1 for s, m in zip(out.stride(), out.shape)):
                raise ValueError("out must not be an expanded tensor")
        if q.numel() == 0:
            return out
        if self._captured or _capturing():
            most = max(self._cap[i] for i in ids)
        elif self._key is not None and self._key == key:
            most = self._most
        else:
            self._settle()
            most = max(self._bound[i] for i in ids)
        size = (_lib._lib or _lib.lib()).ress_kv_attend_workspace_size(self._handle, B, Hq, n, most)
        work = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        P = _lib.ptr
        self._call("ress_kv_attend", self._handle, P(q), *qs, B, Hq, n, P(slot_t), P(lens_t), 1 if causal else 0, scale,
                   most, P(out), *os, P(work), size)
        return out
