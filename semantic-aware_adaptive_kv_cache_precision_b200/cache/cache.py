"""The cache of live sequences.

Every live sequence holds a slot. Cache entries (one per layer call that writes
a cache) are sorted into groups by what they need:

* entries with the same `KVNeed` (heads, key and value widths, window, type) form a KV
  group with storage of its own: `keys` [entries, blocks, kv_heads, 64, head_dim] and
  `values` [..., value_dim], a pool of blocks, and for every slot the list of blocks that hold
  its positions 0-63, 64-127, ... A group with a window gives a sequence's
  blocks back as soon as every position in them has fallen out of the window.
* every entry with a `StateNeed` has a tensor [slots, *shape]: state of fixed
  size per sequence, zeroed when a slot is taken.
* a sequence that is forked (`SequenceCache.fork`) shares its full blocks with the new ones: a
  block goes back to its pool when the last sequence that lists it lets go of it.
* an entry with a `MultiNeed` holds one of the above for each of its parts (an attention
  layer that also keeps a little running state beside its keys and values).

Each sequence has its own length. Storage is sized by `max_tokens`, the most
positions that live sequences hold at any time with each sequence's count
rounded up to a multiple of 64. The reference's caches hold one sequence
(`src/microinfer/model.py:95-132, 147-286`); slots, groups and state are this
library's own.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from .. import ops
from ..errors import allocate
from .allocator import CacheFull, Pool
from .needs import KVNeed, MultiNeed, StateNeed

BLOCK = 64

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int32": torch.int32}


@dataclass
class EntryView:
    """What one layer call sees of the cache during a step."""
    need: object
    keys: torch.Tensor | None = None          # [blocks, kv_heads, 64, head_dim]
    values: torch.Tensor | None = None        # [blocks, kv_heads, 64, value_dim]; None if 0
    block_table: torch.Tensor | None = None   # int32 [B, max_blocks], this step's sequences
    state: torch.Tensor | None = None         # [slots, *shape]; index with the step's slots
    group: int = -1
    parts: list | None = None                 # a `MultiNeed`'s views, one for each of its needs


class KVGroup:
    def __init__(self, need: KVNeed, entries: list[int], blocks: int, max_blocks_per_seq: int,
                 max_slots: int, dtype: torch.dtype, device):
        self.need, self.entries = need, entries
        self.pool = Pool(blocks, "cache block")
        self.holders = np.zeros(blocks, dtype=np.int32)     # sequences that list each block
        # moves whenever the sequences that share blocks of this group may have changed
        self.sharing = 0
        if need.dtype is not None:
            if need.dtype not in _DTYPES:
                raise TypeError(f"{need!r}: dtype must be one of {sorted(_DTYPES)} or None")
            dtype = _DTYPES[need.dtype]
        self.dtype, self.device = dtype, device
        self.keys, self.values = self.storage(blocks)
        self.max_blocks_per_seq = max_blocks_per_seq
        # host copy of every slot's block list; -1 = no block
        self.tables = np.full((max_slots, max_blocks_per_seq), -1, dtype=np.int32)

    def storage(self, blocks: int):
        """Zeroed (keys, values) of `blocks` blocks; values None where the need has none."""
        def zeros(width):
            shape = (len(self.entries), max(blocks, 1), self.need.kv_heads, BLOCK, width)
            count = int(np.prod(shape))
            return allocate(lambda: torch.zeros(shape, dtype=self.dtype, device=self.device),
                            f"a cache of {blocks} blocks of {BLOCK} positions for "
                            f"{len(self.entries)} layer(s)", count * self.dtype.itemsize)

        return zeros(self.need.head_dim), (None if self.need.value_width == 0
                                           else zeros(self.need.value_width))

    @property
    def tensors(self) -> list:
        return [t for t in (self.keys, self.values) if t is not None]


class SequenceCache:
    """Slots, blocks, lengths and per-sequence state of all live sequences."""

    def __init__(self, needs: list, max_tokens: int, max_positions: int, dtype: torch.dtype,
                 device, max_slots: int | None = None, poison_freed: bool = False):
        if max_tokens <= 0:
            raise ValueError(f"max_tokens must be positive, got {max_tokens}")
        self.dtype, self.device = dtype, torch.device(device)
        self.blocks = -(-max_tokens // BLOCK)
        self.max_tokens = self.blocks * BLOCK
        self.max_positions = max_positions
        self.max_seq_len = min(max_positions, self.max_tokens)
        self.max_blocks_per_seq = -(-self.max_seq_len // BLOCK)
        self.max_slots = max_slots if max_slots is not None else min(self.blocks, 1024)
        self.poison_freed = poison_freed
        self.slots = Pool(self.max_slots, "sequence slot")
        self.lengths = np.zeros(self.max_slots, dtype=np.int64)
        self.needs = list(needs)
        self.groups: list[KVGroup] = []
        self.entry_group: dict[int, tuple[int, int]] = {}     # entry -> (group, index in group)
        self.states: dict[int, torch.Tensor] = {}
        by_need: dict[KVNeed, list] = {}

        def place(key, need):
            # `key`: the entry's number, or (its key, part) for a part of a `MultiNeed`
            if isinstance(need, KVNeed):
                by_need.setdefault(need, []).append(key)
            elif isinstance(need, StateNeed):
                shape = (self.max_slots,) + tuple(need.shape)
                self.states[key] = allocate(
                    lambda: torch.zeros(shape, dtype=_DTYPES[need.dtype], device=device),
                    f"the per-sequence state of cache entry {key}",
                    int(np.prod(shape)) * _DTYPES[need.dtype].itemsize)
            elif isinstance(need, MultiNeed):
                for i, part in enumerate(need.parts):
                    place((key, i), part)
            elif need is not None:
                raise TypeError(f"cache entry {key}: unknown need {need!r}")

        for entry, need in enumerate(self.needs):
            place(entry, need)
        for need, entries in by_need.items():
            g = len(self.groups)
            self.groups.append(KVGroup(need, entries, self.blocks, self.max_blocks_per_seq,
                                       self.max_slots, dtype, device))
            for i, entry in enumerate(entries):
                self.entry_group[entry] = (g, i)
        # holders beyond the first, over all blocks (0: no block is listed twice)
        self._shared = 0
        # first position whose block a window group still holds, per (group, slot)
        self._front = [np.zeros(self.max_slots, dtype=np.int64) for _ in self.groups]

    # -- sizes --------------------------------------------------------------

    @property
    def nbytes(self) -> int:
        total = sum(t.numel() * t.element_size() for g in self.groups
                    for t in (g.keys, g.values) if t is not None)
        return total + sum(s.numel() * s.element_size() for s in self.states.values())

    # -- slots --------------------------------------------------------------

    def open(self, count: int = 1) -> list[int]:
        """Take `count` slots (all or none) for sequences of length 0."""
        slots = self.slots.take(count)
        for s in slots:
            self.lengths[s] = 0
            for g, group in enumerate(self.groups):
                group.tables[s, :] = -1
                self._front[g][s] = 0
        if slots and self.states:
            index = torch.as_tensor(slots, dtype=torch.long, device=self.device)
            for state in self.states.values():
                state.index_fill_(0, index, 0)
        return slots

    def close(self, slots) -> None:
        """End sequences: their blocks and slots go back to the pools."""
        slots = list(slots)
        for s in slots:
            if s not in self.slots._held:
                raise RuntimeError(f"slot {s} is not held (closed twice, or never opened)")
        for s in slots:
            for g, group in enumerate(self.groups):
                row = group.tables[s]
                self._release(group, [int(b) for b in row[row >= 0]])
                row[:] = -1
            self.lengths[s] = 0
        self.slots.give_back(slots)

    def _release(self, group: KVGroup, blocks: list[int]) -> None:
        """A sequence lets go of `blocks`; those that no other sequence lists go back to the pool."""
        if not blocks:
            return
        group.holders[blocks] -= 1
        if self._shared:
            kept = len(blocks)
            blocks = [b for b in blocks if group.holders[b] == 0]
            kept -= len(blocks)
            self._shared -= kept
            group.sharing += kept > 0
            if not blocks:
                return
        if self.poison_freed and group.keys.is_floating_point():
            index = torch.as_tensor(blocks, dtype=torch.long, device=self.device)
            group.keys.index_fill_(1, index, float("nan"))
            if group.values is not None:
                group.values.index_fill_(1, index, float("nan"))
        group.pool.give_back(blocks)

    # -- forks ----------------------------------------------------------------

    @property
    def shares_blocks(self) -> bool:
        """Whether some block is listed by more than one sequence."""
        return self._shared > 0

    def _copy(self, tensors, src, dst, **how) -> None:
        if self.device.type == "cuda":
            ops.copy_blocks(tensors, src, dst, **how)
            return
        # (a cache whose tensors lie on the host: the bookkeeping's tests)
        into = how.get("into") or tensors
        for t, u in zip(tensors, into):
            if how.get("axis", 1) == 0:
                u[dst] = t[src]
            else:
                u[:, dst, :, :how.get("rows") or BLOCK] = t[:, src, :, :how.get("rows") or BLOCK]

    def fork(self, slot: int, count: int = 1) -> list[int]:
        """`count` new sequences that begin with everything the sequence in `slot` has: its length, its
        blocks and its state. Blocks whose 64 positions are all filled are shared (a sequence writes
        behind its length only), the last, partly filled one and the state are copied. All or nothing: if
        slots or blocks are lacking, nothing changes."""
        if slot not in self.slots._held:
            raise RuntimeError(f"slot {slot} is not held (closed, or never opened)")
        if count < 0:
            raise ValueError(f"cannot fork {count} sequences")
        length = int(self.lengths[slot])
        full, rows = divmod(length, BLOCK)
        for group in self.groups:
            if rows and group.pool.free < count:
                raise CacheFull(f"{count} cache block(s) of {BLOCK} positions needed, {group.pool.free} of "
                                f"{group.pool.size} free; nothing was taken")
        new = self.slots.take(count)
        if not count:
            return new
        for g, group in enumerate(self.groups):
            row = group.tables[slot]
            common = row[:full]
            listed = common[common >= 0]
            group.holders[listed] += count
            group.sharing += 1
            self._shared += count * len(listed)
            group.tables[new] = -1
            group.tables[new, :full] = common
            self._front[g][new] = self._front[g][slot]
            if rows:
                own = group.pool.take(count)
                group.holders[own] = 1
                group.tables[new, full] = own
                self._copy(group.tensors, [int(row[full])] * count, own, rows=rows)
        self.lengths[new] = length
        if self.states:
            by_type = list(self.states.values())
            self._copy(by_type, [slot] * count, new, axis=0)
        return new

    # -- another size ---------------------------------------------------------

    def sizes_for(self, max_tokens: int) -> tuple:
        """(blocks of every pool, longest sequence) of a cache of `max_tokens` positions; `CacheFull` where what is
        held now would not fit it."""
        if max_tokens <= 0:
            raise ValueError(f"max_tokens must be positive, got {max_tokens}")
        blocks = -(-max_tokens // BLOCK)
        longest = min(self.max_positions, blocks * BLOCK)
        width = -(-longest // BLOCK)
        for group in self.groups:
            if group.pool.held > blocks:
                raise CacheFull(f"{group.pool.held} cache blocks are held, {blocks} would not hold them; "
                                "nothing was changed")
        for s in self.slots._held:
            if self.lengths[s] > longest or any((group.tables[s, width:] >= 0).any() for group in self.groups):
                raise CacheFull(f"a sequence of {int(self.lengths[s])} positions does not fit a cache of "
                                f"{longest} per sequence; nothing was changed")
        return blocks, longest

    def resize(self, max_tokens: int, max_slots: int | None = None) -> None:
        """Give every pool room for `max_tokens` positions (rounded up to blocks) while sequences live:
        held blocks are moved into new storage, one behind the other in the order of their numbers, and the
        old storage is given up. `max_slots`: as many slots at least (they never become fewer). All or
        nothing: `CacheFull` where the held blocks, or a sequence's length, do not fit; `OutOfDeviceMemory`
        where the device has no room for old and new storage together."""
        blocks, longest = self.sizes_for(max_tokens)
        width = -(-longest // BLOCK)
        slots = max(self.max_slots, max_slots or 0)
        storage = [group.storage(blocks) for group in self.groups]
        states = self.states if slots == self.max_slots else {
            key: allocate(lambda: torch.zeros((slots,) + tuple(t.shape[1:]), dtype=t.dtype, device=t.device),
                          f"the per-sequence state of cache entry {key}", slots * t[0].numel() * t.element_size())
            for key, t in self.states.items()}
        for group, new in zip(self.groups, storage):
            held = sorted(group.pool._held)
            self._copy(group.tensors, held, list(range(len(held))), into=[t for t in new if t is not None])
        if states is not self.states:
            live = sorted(self.slots._held)
            self._copy(list(self.states.values()), live, live, into=list(states.values()), axis=0)
        # (from here on nothing can fail)
        for group, (keys, values) in zip(self.groups, storage):
            held = sorted(group.pool._held)
            place = np.full(group.pool.size + 1, -1, dtype=np.int32)       # (the last: -1 stays -1)
            place[held] = np.arange(len(held), dtype=np.int32)
            tables = np.full((slots, width), -1, dtype=np.int32)
            kept = min(width, group.max_blocks_per_seq)
            tables[:self.max_slots, :kept] = place[group.tables[:, :kept]]
            holders = np.zeros(blocks, dtype=np.int32)
            holders[:len(held)] = group.holders[held]
            group.pool = Pool(blocks, "cache block")
            group.pool.take(len(held))
            group.keys, group.values = keys, values
            group.tables, group.holders, group.max_blocks_per_seq = tables, holders, width
            group.sharing += 1
        more = slots - self.max_slots
        if more:
            self.states = states
            self.slots.grow(slots)
            self.lengths = np.concatenate([self.lengths, np.zeros(more, dtype=np.int64)])
            self._front = [np.concatenate([f, np.zeros(more, dtype=np.int64)]) for f in self._front]
            self.max_slots = slots
        self.blocks, self.max_tokens = blocks, blocks * BLOCK
        self.max_seq_len, self.max_blocks_per_seq = longest, width

    # -- growth -------------------------------------------------------------

    def reserve(self, slots, new_lengths) -> None:
        """Make room for every sequence `slots[i]` to reach `new_lengths[i]`
        positions. All or nothing: if any group lacks blocks, or a sequence would
        pass the longest length the cache takes, nothing changes."""
        plans = []
        for g, group in enumerate(self.groups):
            want = []
            for s, n in zip(slots, new_lengths):
                if n > self.max_seq_len:
                    raise CacheFull(f"a sequence of {n} positions exceeds the {self.max_seq_len} "
                                    "that this cache takes per sequence; nothing was taken")
                first = int(self._front[g][s]) // BLOCK
                last = -(-int(n) // BLOCK)
                kept = -(-int(group.need.keep_first or 0) // BLOCK)     # never given back
                missing = [b for b in list(range(min(kept, first, last)))
                           + list(range(first, last)) if group.tables[s, b] < 0]
                want.append((s, missing))
            total = sum(len(m) for _, m in want)
            if total > group.pool.free:
                raise CacheFull(f"{total} cache block(s) of {BLOCK} positions needed, "
                                f"{group.pool.free} of {group.pool.size} free; nothing was taken")
            plans.append((group, want))
        for group, want in plans:
            for s, missing in want:
                for b, block in zip(missing, group.pool.take(len(missing))):
                    group.tables[s, b] = block
                    group.holders[block] = 1

    def advance(self, slots, new_lengths) -> None:
        """Record the new lengths after a step; window groups give back the blocks
        whose positions no later query can see."""
        for s, n in zip(slots, new_lengths):
            self.lengths[s] = n
            for g, group in enumerate(self.groups):
                w = group.need.window
                if not w:
                    continue
                first_seen = max(0, int(n) - w + 1)       # oldest position the next query sees
                keep_from = first_seen // BLOCK
                old = int(self._front[g][s]) // BLOCK
                if keep_from > old:
                    row = group.tables[s]
                    # (the blocks of the first `keep_first` positions stay where they are)
                    old = max(old, -(-int(group.need.keep_first or 0) // BLOCK))
                    gone = [int(b) for b in row[old:keep_from] if b >= 0]
                    row[old:keep_from] = -1
                    self._release(group, gone)
                    self._front[g][s] = keep_from * BLOCK

    # -- what a step sees -----------------------------------------------------

    def tables_for(self, slots) -> list[np.ndarray]:
        """For each KV group, the block lists of `slots` as int32 [B, max_blocks]."""
        index = np.asarray(list(slots), dtype=np.int64)
        return [group.tables[index] for group in self.groups]

    def entry_view(self, entry, device_tables: list, need=None) -> EntryView:
        need = self.needs[entry] if need is None else need
        if isinstance(need, MultiNeed):
            return EntryView(need, parts=[self.entry_view((entry, i), device_tables, part)
                                          for i, part in enumerate(need.parts)])
        if isinstance(need, KVNeed):
            g, i = self.entry_group[entry]
            group = self.groups[g]
            return EntryView(need, group.keys[i],
                             None if group.values is None else group.values[i],
                             device_tables[g], None, g)
        if isinstance(need, StateNeed):
            return EntryView(need, state=self.states[entry])
        return EntryView(need)

    def check(self) -> None:
        """Bookkeeping invariants: no slot or block lost, held twice or freed twice."""
        self.slots.check()
        for group in self.groups:
            group.pool.check()
            listed = group.tables[group.tables >= 0].tolist()
            counts = np.bincount(np.asarray(listed, dtype=np.int64), minlength=len(group.holders))
            if (counts != group.holders).any():
                raise RuntimeError("a cache block is listed for more or fewer places than it counts")
            for s in range(self.max_slots):
                row = group.tables[s][group.tables[s] >= 0]
                if len(np.unique(row)) != len(row):
                    raise RuntimeError("a cache block is listed for two places")
            # (a block that sequences share holds the same positions of each)
            if len(np.unique(np.argwhere(group.tables >= 0)[:, 1] * (len(group.holders) + 1)
                             + group.tables[group.tables >= 0])) != len(set(listed)):
                raise RuntimeError("a cache block is listed for two places")
            if set(listed) != group.pool._held:
                raise RuntimeError("held blocks and listed blocks differ: "
                                   f"{sorted(group.pool._held ^ set(listed))}")
            for s in range(self.max_slots):
                if s not in self.slots._held and (group.tables[s] >= 0).any():
                    raise RuntimeError(f"free slot {s} still lists blocks")
        if self._shared != sum(int(np.maximum(g.holders - 1, 0).sum()) for g in self.groups):
            raise RuntimeError("the count of shared blocks is wrong")
