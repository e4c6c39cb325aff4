"""The cache of a model: keys and values per layer run, per-sequence state of
fixed size, and the slots that tie both to sequences.

What a mixer needs is a *request*: `KVRequest` (keys and values of so many
heads of such a size, all of them or a window) or `StateRequest` (a record of
fixed shape per sequence).  Runs whose KV requests are equal form a *group*
with storage of its own -- its own pages, page pool and block table -- so that
layers that keep every key and layers that keep a window do not share storage.

Storage of a group: ``pages[entry, page, 0|1, kv_head, token(64), channel]``
(keys at 0, values at 1; a request with ``planes=1`` has the key plane only and
its view hands out the key plane as the value plane too: a mixer whose values
are a part of what it stores as keys).  A request whose values have a size of
their own (``value_dim``) keeps, per page, the key block ``[kv_head, 64,
head_dim]`` and behind it the value block ``[kv_head, 64, value_dim]``; both
planes still share one page stride and one block table.  ``block_table[slot, i]`` is the page holding tokens
``[64*i, 64*i+64)`` of the sequence in `slot`.  A sequence holds
ceil(length/64) pages per group -- a group that keeps a window gives back, as
the sequence grows, the pages that have slid out of it; a group whose keys are seen
within stretches of ``chunk`` positions gives back the pages that lie wholly
before the stretch of the next token -- and pages and the
slot return to the free lists when the sequence is closed, and are handed out
again.

A cache with ``kv_format="e4m3"`` holds its keys and values in 8 bits: code * scale, the codes
in e4m3, one power of two as scale for each block of 64 rows (a page) of one head, keys and values apart.
A group's storage is then an `E4M3Storage`: ``k[entry, page, kv_head, token(64), channel]``, ``v[entry, page,
kv_head, channel, token(64)]`` and ``scales[entry, page, 0|1, kv_head]`` (csrc/e4m3.cuh has the codes).  Mixers say
which of their requests such a cache can serve (`KVRequest.e4m3`).  With a `KeepRule` beside it the cache also
gathers every row's attention weight, and a sequence that holds ``budget + slack`` rows is cut back to ``budget``:
its newest rows and the heaviest of the others, chosen per layer run and head (`Cache.evict`).  From then on a sequence's
length (its positions) and the rows it holds are two numbers: position p lies in row p - dropped.

The reference keeps one growing slice (CPU) or one 2048-position buffer (GPU)
per layer for its single sequence (model/llama.go:984-985,1017-1029;
model/gpu_forward.go:477-496); per-layer widths for layers that reuse another
layer's cache are in model/kv_staging.go:11-54.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from ..kernels import ops
from .pages import CacheFull, CacheMisuse, PagePool, SlotTable

PAGE_TOKENS = 64


@dataclass(frozen=True)
class KVRequest:
    n_kv_heads: int
    head_dim: int
    window: Optional[int] = None      # None: every key is kept
    planes: int = 2                   # 2: keys and values; 1: keys only (the values are a part of the key rows)
    value_dim: Optional[int] = None   # channels of a stored value; None: head_dim
    chunk: Optional[int] = None       # keys are seen within stretches of so many positions (None: not)
    # whether the mixer's kernels take an e4m3 cache; requests that differ in nothing else share storage
    e4m3: bool = field(default=False, compare=False)

    @property
    def first_needed(self):
        """A function of the next token's position: the first position it still sees."""
        def lo(position: int) -> int:
            first = 0
            if self.window is not None:
                first = max(first, position - self.window + 1)
            if self.chunk is not None:
                first = max(first, position - position % self.chunk)
            return first
        return lo

    @property
    def forgets(self) -> bool:
        return self.window is not None or self.chunk is not None


@dataclass(frozen=True)
class KeepRule:
    """How many rows a sequence of an evicting cache keeps: once it holds `budget` + `slack` after a step, it is cut
    back to `budget`, its `recent` newest among them."""
    budget: int
    recent: int
    slack: int = PAGE_TOKENS

    def __post_init__(self):
        if self.budget < 1 or not 0 <= self.recent <= self.budget or self.slack < 1:
            raise ValueError(f"a keep rule needs a positive budget, 0 <= recent <= budget and a positive slack, got "
                             f"budget {self.budget}, recent {self.recent}, slack {self.slack}")

    @property
    def most(self) -> int:
        """Rows a sequence holds at most between steps of one token."""
        return self.budget + self.slack


@dataclass(frozen=True)
class StateRequest:
    name: str
    shape: Tuple[int, ...]
    dtype: str = "float32"            # "float32" | "bfloat16" | "int32"


Request = Union[KVRequest, StateRequest]
_STATE_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int32": torch.int32}


KV_FORMATS = (None, "e4m3")


class KVEntryView:
    """What a kernel needs to address one run's keys and values."""
    format: Optional[str] = None
    __slots__ = ("k", "v", "page_stride", "block_table", "table_stride", "n_kv_heads", "head_dim",
                 "window", "value_dim", "chunk")

    def __init__(self, k, v, block_table, n_kv_heads, head_dim, window, value_dim=None, chunk=None):
        self.k, self.v = k, v
        self.value_dim = head_dim if value_dim is None else value_dim     # width of a row of the value plane
        self.chunk = chunk
        self.page_stride = k.stride(0)
        self.block_table = block_table
        self.table_stride = block_table.stride(0)
        self.n_kv_heads, self.head_dim, self.window = n_kv_heads, head_dim, window


def _check_e4m3(k, v, scales, block_table, weights, dropped, lead: int) -> None:
    """Shapes, types and layout of an e4m3 cache's tensors; `lead`: axes ahead of the heads."""
    if k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
        raise ValueError(f"an e4m3 cache holds float8_e4m3fn, not {k.dtype} and {v.dtype}")
    if k.dim() != lead + 3 or k.shape[-2] != PAGE_TOKENS:
        raise ValueError(f"keys must be [..., page, head, {PAGE_TOKENS}, channel], got {tuple(k.shape)}")
    pages, n_kv, hd = k.shape[:lead], k.shape[-3], k.shape[-1]
    if tuple(v.shape) != tuple(pages) + (n_kv, hd, PAGE_TOKENS):
        raise ValueError(f"values must be {tuple(pages) + (n_kv, hd, PAGE_TOKENS)}, got {tuple(v.shape)}")
    if scales.dtype != torch.float32 or tuple(scales.shape) != tuple(pages) + (2, n_kv):
        raise ValueError(f"scales must be float32 {tuple(pages) + (2, n_kv)}, got {scales.dtype} {tuple(scales.shape)}")
    if weights is not None and (weights.dtype != torch.float32 or tuple(weights.shape) != tuple(pages) + (n_kv, PAGE_TOKENS)):
        raise ValueError(f"weights must be float32 {tuple(pages) + (n_kv, PAGE_TOKENS)}, got {weights.dtype} {tuple(weights.shape)}")
    for name, t in (("keys", k), ("values", v), ("scales", scales), ("weights", weights)):
        if t is None:
            continue
        inside = t.shape[lead:]
        if t.device != k.device or t.stride()[lead:] != torch.empty(inside, device="meta").stride():
            raise ValueError(f"the {name} of a page must lie in one piece, on the keys' device")
        if t.element_size() == 1 and (t.data_ptr() % 16 or any(st % 16 for st in t.stride()[:lead])):
            raise ValueError(f"the {name} of a page must start on a 16-byte boundary")
        if t is weights and (t.data_ptr() % 16 or any(st % 4 for st in t.stride()[:lead])):
            raise ValueError("the weights of a page must start on a 16-byte boundary")
    if (block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1 or block_table.stride(0) < block_table.shape[1]
            or block_table.device != k.device):
        raise ValueError("the block table must be int32 [slots, pages of a sequence], row by row, on the keys' device")
    if dropped is not None and (dropped.dtype != torch.int32 or not dropped.is_contiguous() or dropped.numel() != block_table.shape[0]
                                or dropped.device != k.device):
        raise ValueError("dropped must be contiguous int32 [slots] on the keys' device")


class _E4M3Pages(ctypes.Structure):
    """The same in C (csrc/e4m3.cuh)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_stride", ctypes.c_longlong), ("v_stride", ctypes.c_longlong),
                ("scales", ctypes.c_void_p), ("scale_stride", ctypes.c_longlong), ("weights", ctypes.c_void_p), ("weight_stride", ctypes.c_longlong),
                ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_int), ("dropped", ctypes.c_void_p), ("n_kv", ctypes.c_int),
                ("hd", ctypes.c_int)]

    @classmethod
    def of(cls, k, v, scales, block_table, weights, dropped):
        """Of tensors as `E4M3KVView` has them, or `E4M3Storage`: of its entry 0."""
        at = k.dim() - 4                                     # the axis of pages
        return cls(k.data_ptr(), v.data_ptr(), k.stride(at), v.stride(at), scales.data_ptr(), scales.stride(at),
                   weights.data_ptr() if weights is not None else None, weights.stride(at) if weights is not None else 0,
                   block_table.data_ptr(), block_table.stride(0), dropped.data_ptr() if dropped is not None else None,
                   k.shape[at + 1], k.shape[at + 3])


class E4M3KVView:
    """What a kernel needs to address one run's keys and values in an e4m3 cache: k [page, head, 64, channel] and v
    [page, head, channel, 64] (float8_e4m3fn), scales [page, 2, head] (float32 powers of two), the block table, and for a cache
    that evicts weights [page, head, 64] (float32) and dropped [slot] (int32, rows evicted so far)."""
    format = "e4m3"
    chunk = None

    def __init__(self, k, v, scales, block_table, window=None, weights=None, dropped=None):
        _check_e4m3(k, v, scales, block_table, weights, dropped, lead=1)
        self.k, self.v, self.scales, self.weights = k, v, scales, weights
        self.block_table, self.dropped, self.window = block_table, dropped, window
        self.n_kv_heads, self.head_dim = k.shape[1], k.shape[3]
        self.value_dim = self.head_dim
        self.page_stride, self.table_stride = k.stride(0), block_table.stride(0)
        self._pages = _E4M3Pages.of(k, v, scales, block_table, weights, dropped)
        self._address = ctypes.addressof(self._pages)

    def address(self) -> int:
        """Where the pointers and strides lie as the kernels take them."""
        return self._address


class E4M3Storage:
    """All runs of one group of an e4m3 cache: the tensors of `E4M3KVView` with an entry axis in front of the pages."""
    format = "e4m3"

    def __init__(self, k, v, scales, block_table, window=None, weights=None, dropped=None):
        _check_e4m3(k, v, scales, block_table, weights, dropped, lead=2)
        self.k, self.v, self.scales, self.weights = k, v, scales, weights
        self.block_table, self.dropped, self.window = block_table, dropped, window
        self.n_kv_heads, self.head_dim = k.shape[2], k.shape[4]
        self._pages = _E4M3Pages.of(k, v, scales, block_table, weights, dropped)
        self._address = ctypes.addressof(self._pages)
        # how far entries are apart: keys, values, scales, weights
        self.entry_strides = (k.stride(0), v.stride(0), scales.stride(0), weights.stride(0) if weights is not None else 0)

    def address(self) -> int:
        """Where entry 0's pointers and strides lie as the kernels take them."""
        return self._address

    def entry(self, i: int) -> E4M3KVView:
        return E4M3KVView(self.k[i], self.v[i], self.scales[i], self.block_table, self.window,
                          self.weights[i] if self.weights is not None else None, self.dropped)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.scales, self.weights) if t is not None)


class CacheHandle:
    """The storage of one schedule entry: `.kv` (or None) and `.state(name)`.
    `writes` is False when the entry reads another entry's storage."""

    def __init__(self, kv: Optional[KVEntryView], states: Dict[str, torch.Tensor], writes: bool):
        self.kv = kv
        self._states = states
        self.writes = writes

    def state(self, name: str) -> torch.Tensor:
        """[n_slots, *shape]; row `slot` belongs to the sequence in that slot."""
        return self._states[name]


class _KVGroup:
    def __init__(self, request: KVRequest, n_entries: int, n_pages: int, n_slots: int,
                 pages_per_seq: int, dtype: torch.dtype, device: torch.device,
                 kv_format: Optional[str] = None, keep: Optional[KeepRule] = None):
        self.request = request
        self.pool = PagePool(n_pages)
        self.e4m3: Optional[E4M3Storage] = None
        if request.planes not in (1, 2):
            raise ValueError(f"a key/value store has 1 or 2 planes, not {request.planes}")
        self.value_dim = request.head_dim if request.value_dim is None else int(request.value_dim)
        if kv_format == "e4m3":
            if request.planes != 2 or self.value_dim != request.head_dim or request.chunk is not None:
                raise ValueError("an e4m3 cache holds keys and values of one size, without stretches")
            # per page: the keys' codes, then the values'
            self.storage = torch.zeros((n_entries, n_pages, 2, request.n_kv_heads * PAGE_TOKENS * request.head_dim),
                                       dtype=torch.uint8, device=device)
        elif self.value_dim != request.head_dim:
            if request.planes != 2:
                raise ValueError("values of a size of their own need a value plane")
            # per page: the key block, then the value block
            self.storage = torch.zeros((n_entries, n_pages, request.n_kv_heads * PAGE_TOKENS *
                                        (request.head_dim + self.value_dim)), dtype=dtype, device=device)
        else:
            self.storage = torch.zeros((n_entries, n_pages, request.planes, request.n_kv_heads, PAGE_TOKENS,
                                        request.head_dim), dtype=dtype, device=device)
        self.table_host = torch.zeros((n_slots, pages_per_seq), dtype=torch.int32)
        self.table = torch.zeros((n_slots, pages_per_seq), dtype=torch.int32, device=device)
        self.pages_of: Dict[int, List[int]] = {}     # slot -> its pages by index; -1: given back (slid out of the window)
        self.dirty: set = set()
        if kv_format == "e4m3":
            r, lead = request, (n_entries, n_pages)
            codes = self.storage.view(torch.float8_e4m3fn)
            self.e4m3 = E4M3Storage(
                codes[:, :, 0].unflatten(2, (r.n_kv_heads, PAGE_TOKENS, r.head_dim)),
                codes[:, :, 1].unflatten(2, (r.n_kv_heads, r.head_dim, PAGE_TOKENS)),
                torch.full(lead + (2, r.n_kv_heads), 2.0 ** -126, dtype=torch.float32, device=device),
                self.table, r.window,
                torch.zeros(lead + (r.n_kv_heads, PAGE_TOKENS), dtype=torch.float32, device=device) if keep else None,
                torch.zeros(n_slots, dtype=torch.int32, device=device) if keep else None)

    def bytes(self) -> int:
        if self.e4m3 is not None:
            return self.e4m3.bytes()
        return self.storage.numel() * self.storage.element_size()

    def view(self, entry: int) -> Union[KVEntryView, E4M3KVView]:
        if self.e4m3 is not None:
            return self.e4m3.entry(entry)
        s = self.storage[entry]
        r = self.request
        if self.value_dim != r.head_dim:
            split = r.n_kv_heads * PAGE_TOKENS * r.head_dim
            k = s[:, :split].view(s.shape[0], r.n_kv_heads, PAGE_TOKENS, r.head_dim)
            v = s[:, split:].view(s.shape[0], r.n_kv_heads, PAGE_TOKENS, self.value_dim)
            return KVEntryView(k, v, self.table, r.n_kv_heads, r.head_dim, r.window, self.value_dim, r.chunk)
        return KVEntryView(s[:, 0], s[:, r.planes - 1], self.table, r.n_kv_heads, r.head_dim, r.window,
                           self.value_dim, r.chunk)


class Cache:
    """`requests[i]` lists what schedule entry i needs; `shared_from[i]` names the
    entry whose key/value storage entry i reads instead of having its own (such
    an entry asks for no keys and values, but may ask for fixed-size state).
    `kv_format` "e4m3" holds keys and values in 8 bits; `keep` beside it evicts (see the module's head)."""

    def __init__(self, requests: Sequence[Sequence[Request]], shared_from: Sequence[Optional[int]],
                 *, max_tokens: int, max_slots: Optional[int] = None, max_position: Optional[int] = None,
                 dtype: torch.dtype, device: Union[str, torch.device],
                 kv_format: Optional[str] = None, keep: Optional[KeepRule] = None):
        if kv_format not in KV_FORMATS:
            raise ValueError(f"kv_format {kv_format!r} is not known; known: {KV_FORMATS}")
        if keep is not None and kv_format != "e4m3":
            raise ValueError("a keep rule needs kv_format='e4m3': other caches gather no attention weights")
        self.kv_format, self.keep = kv_format, keep
        self.device = torch.device(device)
        self.dtype = dtype
        if max_tokens <= 0:
            raise ValueError("max_tokens must be positive")
        self.n_pages = (max_tokens + PAGE_TOKENS - 1) // PAGE_TOKENS
        self.max_tokens = self.n_pages * PAGE_TOKENS
        self.n_slots = max_slots if max_slots is not None else min(self.n_pages, 1024)
        per_seq = self.n_pages
        if max_position is not None:
            per_seq = min(per_seq, (max_position + PAGE_TOKENS - 1) // PAGE_TOKENS)
        self.pages_per_seq = max(1, per_seq)
        # the longest sequence, in tokens: what the pages of one sequence hold, and no
        # more than the model's own longest position where one is given
        self.max_sequence = self.pages_per_seq * PAGE_TOKENS
        if max_position is not None:
            self.max_sequence = min(self.max_sequence, int(max_position))
        # rows a sequence may hold; a cache that evicts takes sequences of any length the model has positions for
        self.max_held = self.max_sequence
        if keep is not None:
            if keep.most > self.pages_per_seq * PAGE_TOKENS:
                raise ValueError(f"a sequence keeps up to {keep.most} rows, the cache holds {self.pages_per_seq * PAGE_TOKENS} of one")
            self.max_held = self.pages_per_seq * PAGE_TOKENS
            self.max_sequence = int(max_position) if max_position is not None else (1 << 31) - 1
        self.slots = SlotTable(self.n_slots)
        self._length = [0] * self.n_slots
        self._dropped = [0] * self.n_slots
        self._flushed: Optional[Tuple[object, object]] = None      # stream of the last copy of block-table rows, and an event behind it
        # what users of the cache keep with it and want gone when it goes (the generation
        # loop: its recorded decode steps); the cache itself never looks inside
        self.attachments: Dict[str, object] = {}

        # group the KV requests
        keys: List[KVRequest] = []
        members: Dict[KVRequest, List[int]] = {}
        for i, reqs in enumerate(requests):
            for r in reqs:
                if isinstance(r, KVRequest):
                    if kv_format == "e4m3" and not r.e4m3:
                        raise ValueError(f"schedule entry {i} asks for keys and values that its mixer does not read from an e4m3 cache")
                    if keep is not None and r.forgets:
                        raise ValueError(f"schedule entry {i} keeps a window of keys: such layers forget by themselves and are not "
                                         f"built together with a keep rule")
                    if r not in members:
                        members[r] = []
                        keys.append(r)
                    members[r].append(i)
        self.groups: List[_KVGroup] = []
        kv_of_entry: Dict[int, Tuple[int, int]] = {}
        for r in keys:
            grp = _KVGroup(r, len(members[r]), self.n_pages, self.n_slots, self.pages_per_seq,
                           dtype, self.device, kv_format, keep)
            for j, i in enumerate(members[r]):
                if i in kv_of_entry:
                    raise ValueError(f"schedule entry {i} asks for two key/value stores")
                kv_of_entry[i] = (len(self.groups), j)
            self.groups.append(grp)

        # fixed-size state
        self._state_tensors: List[torch.Tensor] = []
        states_of_entry: Dict[int, Dict[str, torch.Tensor]] = {}
        for i, reqs in enumerate(requests):
            for r in reqs:
                if isinstance(r, StateRequest):
                    if r.dtype not in _STATE_DTYPES:
                        raise ValueError(f"state dtype {r.dtype!r} is not supported")
                    t = torch.zeros((self.n_slots,) + tuple(r.shape), dtype=_STATE_DTYPES[r.dtype],
                                    device=self.device)
                    states_of_entry.setdefault(i, {})[r.name] = t
                    self._state_tensors.append(t)

        self.handles: List[CacheHandle] = []
        for i in range(len(requests)):
            src = shared_from[i]
            owner = i if src is None else src
            kv = None
            if owner in kv_of_entry:
                g, j = kv_of_entry[owner]
                kv = self.groups[g].view(j)
            # an entry that reads another entry's keys and values may still keep state of its own
            states = dict(states_of_entry.get(owner, {}))
            states.update(states_of_entry.get(i, {}))
            self.handles.append(CacheHandle(kv, states, writes=src is None))

    # ------------------------------------------------------------ sequences
    def open_sequence(self) -> int:
        """A free slot with length 0 and zeroed fixed-size state."""
        slot = self.slots.alloc()
        self._length[slot] = self._dropped[slot] = 0
        for grp in self.groups:
            grp.pages_of[slot] = []
            if self.keep is not None:
                grp.e4m3.dropped[slot].zero_()
        for t in self._state_tensors:
            t[slot].zero_()
        return slot

    def close_sequence(self, slot: int) -> None:
        if not self.slots.is_held(slot):
            raise CacheMisuse(f"slot {slot} is closed but is not open")
        for grp in self.groups:
            grp.pool.free([p for p in grp.pages_of.pop(slot) if p >= 0], slot)
        self._length[slot] = self._dropped[slot] = 0
        self.slots.free(slot)

    def length(self, slot: int) -> int:
        """Tokens of the sequence so far: the next one's position."""
        return self._length[slot]

    def held(self, slot: int) -> int:
        """Rows the sequence has in the cache: its length, less what has been evicted."""
        return self._length[slot] - self._dropped[slot]

    def _pages_for(self, slot: int, new_length: int) -> int:
        """Pages of a sequence grown to `new_length`; refuses one the cache cannot hold."""
        rows = new_length - self._dropped[slot]
        if new_length > self.max_sequence or rows > self.max_held:
            raise CacheFull(f"a sequence of {new_length} tokens exceeds the longest the cache "
                            f"holds ({self.max_sequence if new_length > self.max_sequence else self.max_held})")
        return (rows + PAGE_TOKENS - 1) // PAGE_TOKENS

    def reserve(self, slot: int, new_length: int) -> None:
        """Make room for the sequence in `slot` to grow to `new_length` tokens."""
        if not self.slots.is_held(slot):
            raise CacheMisuse(f"slot {slot} is not open")
        need = self._pages_for(slot, new_length)
        for grp in self.groups:
            have = grp.pages_of[slot]
            if need > len(have):
                if need - len(have) > grp.pool.n_free:
                    raise CacheFull(f"the cache is full: growing a sequence to {new_length} tokens "
                                    f"needs {need - len(have)} more pages of 64 tokens, "
                                    f"{grp.pool.n_free} of {grp.pool.n_pages} are free")
        for grp in self.groups:
            have = grp.pages_of[slot]
            if need > len(have):
                new = grp.pool.alloc(need - len(have), slot)
                grp.table_host[slot, len(have):need] = torch.tensor(new, dtype=torch.int32)
                have.extend(new)
                grp.dirty.add(slot)

    def reserve_many(self, wanted: Sequence[Tuple[int, int]]) -> None:
        """`reserve` for several (slot, new_length) pairs: all of them or none."""
        for grp in self.groups:
            need = 0
            for slot, new_length in wanted:
                if not self.slots.is_held(slot):
                    raise CacheMisuse(f"slot {slot} is not open")
                need += max(0, self._pages_for(slot, new_length) - len(grp.pages_of[slot]))
            if need > grp.pool.n_free:
                raise CacheFull(f"the cache is full: this step needs {need} more pages of 64 tokens, "
                                f"{grp.pool.n_free} of {grp.pool.n_pages} are free")
        for slot, new_length in wanted:
            self.reserve(slot, new_length)

    def advance(self, slot: int, n_tokens: int) -> None:
        """Record that `n_tokens` more tokens of the sequence are in the cache."""
        new_length = self._length[slot] + n_tokens
        for grp in self.groups:
            if new_length - self._dropped[slot] > len(grp.pages_of[slot]) * PAGE_TOKENS:
                raise CacheMisuse(f"slot {slot} advanced to {new_length} tokens without reserved pages")
        self._length[slot] = new_length
        # A group that keeps a window gives back the pages no later token can see: the next
        # token, at position new_length, reaches back to new_length - window + 1 (to the
        # start of its stretch, for keys seen within stretches).  Their
        # table entries stay as they are; no kernel reads a page before a window's first.
        for grp in self.groups:
            if not grp.request.forgets:
                continue
            have = grp.pages_of[slot]
            gone = [i for i in range(min(len(have), grp.request.first_needed(new_length) // PAGE_TOKENS)) if have[i] >= 0]
            if gone:
                grp.pool.free([have[i] for i in gone], slot)
                for i in gone:
                    have[i] = -1

    def truncate(self, slot: int, new_length: int) -> None:
        """Forget the tokens after `new_length` (their pages stay with the sequence).
        Keys and values are addressed by position, so a shorter length is all it
        takes (the reference's rollback does the same: runtime/kv/staging.go:35-68).
        A record of fixed size has already absorbed the tokens to be forgotten and
        cannot give them back: a cache that holds such state refuses, since a shorter
        length beside an unchanged record would be silently wrong."""
        if self._state_tensors and new_length != self._length[slot]:
            raise CacheMisuse("this cache holds per-sequence state of fixed size, which cannot be "
                              "rolled back by shortening a length; close the sequence and run it again")
        if self.keep is not None and new_length != self._length[slot]:
            raise CacheMisuse("this cache gathers attention weights, which cannot be rolled back by shortening a length; "
                              "close the sequence and run it again")
        if not 0 <= new_length <= self._length[slot]:
            raise CacheMisuse(f"cannot truncate slot {slot} from {self._length[slot]} to {new_length}")
        for grp in self.groups:
            if grp.request.forgets and any(p < 0 for p in grp.pages_of[slot][grp.request.first_needed(new_length) // PAGE_TOKENS:
                                                                         (new_length + PAGE_TOKENS - 1) // PAGE_TOKENS]):
                raise CacheMisuse(f"slot {slot} cannot go back to {new_length} tokens: a layer that keeps a window "
                                  f"or a stretch of keys has given back pages that length would need")
        self._length[slot] = new_length

    def evict(self, slots: Sequence[int], budget: Optional[int] = None, recent: Optional[int] = None) -> List[torch.Tensor]:
        """Cut the sequences in `slots` back to `budget` rows (default: the keep rule's), on the current stream, and give back
        the pages that leaves empty.  A sequence that holds no more is left alone.  Returns, per group, what
        `ops.kv_evict_e4m3` returns: the former row of every row kept."""
        if self.keep is None:
            raise CacheMisuse("this cache gathers no attention weights to evict by: make it with a keep rule")
        budget = self.keep.budget if budget is None else int(budget)
        recent = min(self.keep.recent, budget) if recent is None else int(recent)
        if len(set(slots)) != len(slots) or not all(self.slots.is_held(s) for s in slots):
            raise CacheMisuse("evict: the slots must be open, each named once")
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError(f"evict: budget {budget} must be positive and recent {recent} between 0 and it")
        held = [self.held(s) for s in slots]
        if not slots:
            return []
        self.flush_tables()
        both = self._sent(torch.tensor([list(slots), held], dtype=torch.int32))
        kept = [ops.kv_evict_e4m3(grp.e4m3, both[0], both[1], max(held), budget, recent) for grp in self.groups]
        pages = (budget + PAGE_TOKENS - 1) // PAGE_TOKENS
        for slot, rows in zip(slots, held):
            if rows <= budget:
                continue
            self._dropped[slot] += rows - budget
            for grp in self.groups:
                have = grp.pages_of[slot]
                grp.pool.free(have[pages:], slot)
                del have[pages:]
        return kept

    def evict_due(self, slots: Sequence[int]) -> None:
        """What the engine calls after a step: cut back the sequences that have reached the keep rule's limit."""
        if self.keep is not None:
            due = [s for s in slots if self.held(s) >= self.keep.most]
            if due:
                self.evict(due)

    def flush_tables(self) -> None:
        """Copy block-table rows that changed on the host to the device, on the current stream; what was copied on another stream before
        is there for this one's next kernels too."""
        stream = torch.cuda.current_stream(self.device) if self.device.type == "cuda" else None
        if self._flushed is not None and self._flushed[0] != stream:
            stream.wait_event(self._flushed[1])
        changed = False
        for grp in self.groups:
            for slot in sorted(grp.dirty):
                grp.table[slot].copy_(self._staged(grp.table_host[slot]), non_blocking=True)
                changed = True
            grp.dirty.clear()
        if changed and stream is not None:
            self._flushed = (stream, stream.record_event())

    def _staged(self, host: torch.Tensor) -> torch.Tensor:
        """What `host` holds now, where a copy to the device does not stop the host: page-locked memory of its own, which PyTorch hands
        out again only once copies from it are done, so `host` may change meanwhile."""
        if self.device.type != "cuda":
            return host
        return torch.empty(host.shape, dtype=host.dtype, pin_memory=True).copy_(host)

    def _sent(self, host: torch.Tensor) -> torch.Tensor:
        return self._staged(host).to(self.device, non_blocking=True)

    # ------------------------------------------------------------ accounting
    def tokens_held(self) -> int:
        """Tokens of capacity that live sequences hold (each rounded up to 64)."""
        if not self.groups:
            return 0
        return max(sum(sum(1 for p in pages if p >= 0) for pages in grp.pages_of.values())
                   for grp in self.groups) * PAGE_TOKENS

    def free_pages(self) -> List[int]:
        return [grp.pool.n_free for grp in self.groups]

    def open_slots(self) -> List[int]:
        return self.slots.held()

    def bytes(self) -> int:
        total = sum(g.bytes() for g in self.groups)
        return total + sum(t.numel() * t.element_size() for t in self._state_tensors)
