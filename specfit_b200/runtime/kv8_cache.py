"""KV cache in 8 bits, optionally bounded by eviction.

``Kv8Cache`` takes the place of ``ReservedCache`` where a long context's keys
and values should leave the GPU's memory to expert slots: whole blocks of
tokens are held as e4m3 codes with a power-of-two scale per block and head
(``ops.kv8_seal``), the open block and the rows of the running pass in bf16
(the tail), a little over half the bytes of a bf16 cache.  ``LeanQwen3Forward``
attends to it with ``ops.kv8_tree_attention``; the reference keeps a bf16
``DynamicCache`` (src/specfit/runtime/eagle3_tree.py:1496-1500).

A block is sealed once the rows after it have been taken back or kept: at the
start of the next pass, or, after a causal pass (a prefill), at once.  Rolling
back is ``crop``; a length inside a sealed block brings the block's rows back
to bf16, exactly what attention saw.

With ``budget`` every pass also adds up the attention weight that each cached
token received, per KV head (``ops.kv8_attention_mass``), and ``evict()`` keeps
the first ``sinks`` tokens, the last ``recent``, and the heaviest of the others
(``ops.kv_keep_heaviest``, ``ops.kv8_compact``).  A weight stays added when the
row that gave it is taken back (a rejected tree row has looked at the context
too).  Only ``LeanQwen3Forward`` adds weights: ``update`` does not see the queries,
and ``evict()`` warns when rows came that way, since zeros decide nothing but age.
Keys carry their rotary positions, so what stays is not recomputed; ``next_position`` is the position
of the next token, ``get_seq_length`` the number of rows held.
"""
from __future__ import annotations

import warnings

import torch
from transformers.cache_utils import DynamicCache, DynamicLayer

from .. import ops


class Kv8Layer(DynamicLayer):
    in_place = True  # rolling back is ``crop``

    def __init__(self, capacity: int, block: int, tail_room: int, scored: bool) -> None:
        super().__init__()
        self._reserve = capacity    # tokens the code buffers hold at first
        self.block = block
        self.tail_room = tail_room  # rows of a pass the tail has room for beside an open block
        self.scored = scored        # attention weights are added up
        self.sealed = 0
        self.tail = 0
        self.mass = None
        self.unscored = False       # rows came through ``update``, which adds no weights
        self._kt = None

    # ------------------------------------------------------------- buffers
    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        if key_states.dtype != torch.bfloat16:
            raise TypeError("the 8-bit cache takes bf16 keys and values")
        if value_states.shape != key_states.shape:
            raise ValueError("keys and values must have one shape")
        self.dtype, self.device = key_states.dtype, key_states.device
        self._b, self._h, _, self._d = key_states.shape
        self.sealed = self.tail = 0
        self._codes = self._code_buffers(self._reserve)
        self._new_tail(self.block + self.tail_room)
        if self.scored:
            self.mass = torch.zeros(self._b, self._h, self.capacity, dtype=torch.float32, device=self.device)
        self.is_initialized = True

    def _code_buffers(self, tokens: int):
        cap = -(-tokens // self.block) * self.block
        shape = (self._b, self._h, cap, self._d)
        return (torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device),
                torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device),
                torch.empty(self._b, self._h, cap // self.block, dtype=torch.float32, device=self.device),
                torch.empty(self._b, self._h, cap // self.block, dtype=torch.float32, device=self.device))

    def _new_tail(self, rows: int) -> None:
        """A tail of ``rows`` rows that holds the present ones."""
        old_k, old_v = self._kt, self._kt is not None and self._vt
        # Zeros: rows that a captured pass has not written yet hold finite values.
        self._kt = torch.zeros(self._b, self._h, rows, self._d, dtype=torch.bfloat16, device=self.device)
        self._vt = torch.zeros_like(self._kt)
        if old_k is not None and self.tail:
            self._kt[:, :, : self.tail].copy_(old_k[:, :, : self.tail])
            self._vt[:, :, : self.tail].copy_(old_v[:, :, : self.tail])

    def _room_for_codes(self, tokens: int) -> None:
        cap = self._codes[0].shape[2]
        if tokens <= cap:
            return
        new = self._code_buffers(max(tokens, 2 * cap))
        for a, b in zip(new, self._codes):
            a[:, :, : b.shape[2]].copy_(b)
        self._codes = new

    def _room_for_mass(self, tokens: int) -> None:
        if self.scored and self.mass.shape[2] < tokens:
            new = torch.zeros(self._b, self._h, max(tokens, 2 * self.mass.shape[2]), dtype=torch.float32,
                              device=self.device)
            new[:, :, : self.mass.shape[2]].copy_(self.mass)
            self.mass = new

    @property
    def capacity(self) -> int:
        """Tokens that fit without a larger buffer."""
        return self._codes[0].shape[2] + self._kt.shape[2] if self._kt is not None else self._reserve

    def layout(self):
        """What a captured pass over this layer reads and writes by address: its
        buffers, and how many rows are codes and tail."""
        return (*self._codes, self._kt, self._vt), self.sealed, self.tail

    # --------------------------------------------------------------- a pass
    def begin(self, rows: int) -> None:
        """Makes room for ``rows`` more rows at tail row ``self.tail``.  What is
        there stays, so its whole blocks are sealed."""
        self.seal()
        if self.tail + rows > self._kt.shape[2]:
            self._new_tail(self.tail + rows)
        self._room_for_mass(self.length + rows)

    def end(self, rows: int) -> None:
        """``rows`` rows were written at the tail's end."""
        if self.scored:
            self.mass[:, :, self.length: self.length + rows] = 0
        self.tail += rows

    def seal(self) -> None:
        """Seals the tail's whole blocks and gives back a larger tail than reserved."""
        n = self.tail // self.block
        if n:
            full = n * self.block
            self._room_for_codes(self.sealed + full)
            ops.kv8_seal(self._kt[:, :, :full], self._vt[:, :, :full], *self._codes,
                         first_block=self.sealed // self.block, block=self.block)
            rest = self.tail - full  # fewer rows than a block: source and target do not meet
            for t in (self._kt, self._vt):
                t[:, :, :rest].copy_(t[:, :, full: full + rest])
            self.sealed += full
            self.tail = rest
        if self._kt.shape[2] > self.block + self.tail_room:
            self._new_tail(self.block + self.tail_room)

    def rows(self, end: int | None = None) -> "ops.Kv8Rows":
        """The cache, or its rows before ``end`` (in the tail), as the kernels read it."""
        tail = self.tail if end is None else end - self.sealed
        return ops.Kv8Rows(*self._codes, self.sealed, self._kt[:, :, :tail], self._vt[:, :, :tail], self.block)

    # ---------------------------------------------- transformers' interface
    @property
    def length(self) -> int:
        return self.sealed + self.tail

    def get_seq_length(self) -> int:
        return self.length if self.is_initialized else 0

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """Appends and returns all rows in bf16 (for models whose attention
        reads them; the lean forward reads the codes)."""
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        if key_states.shape[:2] != (self._b, self._h) or key_states.shape != value_states.shape:
            raise ValueError("batch or head count differs from the cache")
        n = key_states.shape[2]
        self.unscored = self.scored
        self.begin(n)
        self._kt[:, :, self.tail: self.tail + n].copy_(key_states)
        self._vt[:, :, self.tail: self.tail + n].copy_(value_states)
        self.end(n)
        return ops.kv8_read(self.rows())

    def crop(self, max_length: int) -> None:
        if max_length < 0:
            max_length = self.get_seq_length() - abs(max_length)
        if self.get_seq_length() <= max_length:
            return
        if max_length < 0:
            raise ValueError("more rows cropped than the cache holds")
        if max_length < self.sealed:  # inside a sealed block: its rows become bf16 again
            keep = max_length // self.block * self.block
            k, v = ops.kv8_read(self.rows(), keep, max_length - keep)
            n = max_length - keep
            self._kt[:, :, :n].copy_(k)
            self._vt[:, :, :n].copy_(v)
            self.sealed, self.tail = keep, n
        else:
            self.tail = max_length - self.sealed

    def keep_tail_rows(self, base: int, positions) -> None:
        """Rows ``base + p`` for p in ``positions`` (ascending) move to ``base,
        base + 1, ...`` and the cache ends after them.  ``base`` lies in the tail."""
        if base < self.sealed:
            raise RuntimeError("rows that are sealed cannot be rearranged")
        at = torch.tensor([base - self.sealed + p for p in positions], dtype=torch.long, device=self.device)
        lo, n = base - self.sealed, len(positions)
        for t in (self._kt, self._vt):
            t[:, :, lo: lo + n] = t.index_select(2, at)  # a copy first: the ranges may overlap
        if self.scored:
            self.mass[:, :, base: base + n] = self.mass.index_select(2, at + self.sealed)
        self.tail = lo + n

    def evict(self, budget: int, sinks: int, recent: int) -> int:
        """Keeps ``budget`` rows; returns how many left."""
        gone = self.length - budget
        if gone <= 0:
            return 0
        keep = ops.kv_keep_heaviest(self.mass, self.length, budget, sinks=sinks, recent=recent)
        full = budget // self.block * self.block
        codes = self._code_buffers(self._codes[0].shape[2])
        kt, vt = torch.zeros_like(self._kt), torch.zeros_like(self._vt)
        mass = torch.zeros_like(self.mass)
        new = ops.Kv8Rows(*codes, full, kt[:, :, : budget - full], vt[:, :, : budget - full], self.block)
        ops.kv8_compact(self.rows(), keep, mass=self.mass, out=new, mass_out=mass)
        self._codes, self._kt, self._vt, self.mass = codes, kt, vt, mass
        self.sealed, self.tail = full, budget - full
        return gone

    def reset(self) -> None:
        self.sealed = self.tail = 0
        self.unscored = False

    def offload(self) -> None:
        raise RuntimeError("the 8-bit cache stays on its device")

    prefetch = offload

    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        self.batch_select_indices(beam_idx.to(self.device))

    def batch_repeat_interleave(self, repeats: int) -> None:
        if self.get_seq_length() > 0:
            self._each(lambda t: t.repeat_interleave(repeats, dim=0))

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        if self.get_seq_length() > 0:
            # Bytes: indexing is not defined for every 8-bit float.
            self._each(lambda t: t.view(torch.uint8)[indices].view(t.dtype) if t.dtype == torch.float8_e4m3fn
                       else t[indices])

    def _each(self, f) -> None:
        self._codes = tuple(f(t) for t in self._codes)
        self._kt, self._vt = f(self._kt), f(self._vt)
        if self.scored:
            self.mass = f(self.mass)
        self._b = self._kt.shape[0]


class Kv8Cache(DynamicCache):
    """``DynamicCache`` whose full-attention layers are ``Kv8Layer``s.

    ``capacity``: tokens of context to reserve as codes; ``block``: tokens of a
    scale (32, 64 or 128); ``tail_room``: rows of the largest pass that is not a
    prefill (a verification tree); ``budget``: tokens that ``evict()`` keeps per
    head (None: nothing is scored or evicted), of them ``sinks`` at the start and
    ``recent`` at the end whatever their weight."""

    def __init__(self, *, config, capacity: int, block: int = 64, tail_room: int = 128, budget: int | None = None,
                 sinks: int = 4, recent: int = 64) -> None:
        if capacity <= 0 or tail_room <= 0:
            raise ValueError("capacity and tail_room must be positive")
        if block not in (32, 64, 128):
            raise ValueError("block must be 32, 64 or 128")
        if budget is not None and (sinks < 0 or recent < 0 or sinks + recent > budget or budget <= 0):
            raise ValueError("sinks + recent must fit into a positive budget")
        super().__init__(config=config)
        if any(type(layer) is not DynamicLayer for layer in self.layers):
            raise ValueError("the 8-bit cache takes full-attention layers only")
        self.layers = [Kv8Layer(capacity, block, tail_room, budget is not None) for _ in self.layers]
        self.budget, self.sinks, self.recent = budget, sinks, recent
        self.dropped = 0  # tokens that evictions took out of each head

    def reset(self) -> None:
        super().reset()
        self.dropped = 0

    @property
    def next_position(self) -> int:
        """Position of the next token: rows held and rows evicted."""
        return self.dropped + self.get_seq_length()

    def evict(self) -> int:
        """Cuts every layer to the budget; returns how many rows each lost (0
        when the cache is within it).  The rows of the last pass must be kept
        ones (after ``compact_tree_cache_`` or ``crop``)."""
        if self.budget is None:
            raise RuntimeError("this cache was made without a budget")
        if not self.layers or not self.layers[0].is_initialized:
            return 0
        if any(layer.unscored and layer.length > self.budget for layer in self.layers):
            warnings.warn("rows appended by update() brought no attention weights: the eviction ranks by what the "
                          "lean forward's passes added, and among equal weights keeps the earlier rows",
                          RuntimeWarning, stacklevel=2)
        gone = [layer.evict(self.budget, self.sinks, self.recent) for layer in self.layers]
        if any(g != gone[0] for g in gone):
            raise RuntimeError("the cache's layers differ in length")
        self.dropped += gone[0]
        return gone[0]

    def set_static(self, offset, reported_length: int = 0) -> None:
        if offset is not None:
            raise RuntimeError("the 8-bit cache has no static mode: its blocks are sealed by the host")
