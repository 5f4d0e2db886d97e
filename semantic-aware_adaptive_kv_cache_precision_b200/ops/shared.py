"""Decode attention over blocks that several sequences list (`csrc/attention_shared.cu`), and the plan
that says which. The plan is worked out on the host from the block lists, when sequences are forked or
end, and serves every layer of every step until the next such change."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib
from ._lib import CACHE_BLOCK, KernelError, call_on, require_cuda, sm_count
from .attention import fast_path_takes

UNIT_ROWS = 128           # most rows (sequences x query heads of one KV head) of a unit of work
MOST_GROUP = 16           # most query heads of one KV head, as in the other tensor-core kernels
LEAST_SCALE = 1e-30       # scales from here to its reciprocal
UNIT_WORDS = 8


def common_runs(tables: np.ndarray, lengths: np.ndarray, reach: np.ndarray) -> list:
    """The block lists cut into runs that one set of sequences lists: [(sequences, first column, end)],
    each column of a sequence below its reach in exactly one. A column counts as shared where it is filled
    (below `lengths`) and names the same block; what it is preceded by does not matter, a sum over
    positions can be cut anywhere."""
    count, width = tables.shape
    full = lengths // CACHE_BLOCK
    columns = -(-reach // CACHE_BLOCK)
    runs = []
    shared_to = np.zeros(count, dtype=np.int64)
    if count > 1 and full.max(initial=0) > 0:
        used = int(full.max())
        # (numbers below every block's for columns that are not filled: each its own)
        ids = tables[:, :used].astype(np.int64)
        filled = np.arange(used)[None, :] < full[:, None]
        ids[~filled] = -1 - np.broadcast_to(np.arange(count)[:, None], ids.shape)[~filled]
        order = np.argsort(ids, axis=0, kind="stable")
        ranked = np.take_along_axis(ids, order, axis=0)
        begins = np.ones_like(ranked, dtype=bool)
        begins[1:] = ranked[1:] != ranked[:-1]
        # the first sequence of each group of equal numbers, given to all of the group
        at = np.maximum.accumulate(np.where(begins, np.arange(count)[:, None], 0), axis=0)
        lead = np.empty_like(order)
        np.put_along_axis(lead, order, np.take_along_axis(order, at, axis=0), axis=0)
        several = ~begins                                 # whether anyone else is in the sequence's group
        several[:-1] |= ~begins[1:]
        crowd = np.empty_like(several)
        np.put_along_axis(crowd, order, several, axis=0)
        changes = [0] + (1 + np.flatnonzero((lead[:, 1:] != lead[:, :-1]).any(axis=0))).tolist() + [used]
        open_runs = {}
        for c0, c1 in zip(changes, changes[1:]):
            now = {}
            together = np.flatnonzero(crowd[:, c0])
            for first in np.unique(lead[together, c0]):
                members = tuple(together[lead[together, c0] == first].tolist())
                now[members] = open_runs.pop(members, c0)
            for members, begin in open_runs.items():
                runs.append((members, begin, c0))
            open_runs = now
        for members, begin in open_runs.items():
            runs.append((members, begin, used))
    # what is left of each sequence: its columns outside the runs it belongs to
    own = [[] for _ in range(count)]
    for members, c0, c1 in runs:
        for b in members:
            own[b].append((c0, c1))
    for b in range(count):
        at = 0
        for c0, c1 in sorted(own[b]) + [(int(columns[b]), int(columns[b]))]:
            if c0 > at:
                runs.append(((b,), at, c0))
            at = max(at, c1)
    return runs


# What a unit of work takes where an SM holds two, in us: to start and end, and a block of keys and values (measured
# at head sizes of 64 and 128: 0.9 to 1.1), with more than NARROW_ROWS rows and with fewer; what a partial's
# trip through memory takes, in us a (sequence, head), and its place in the sum over a sequence's partials.
WIDE_US, NARROW_US, NARROW_ROWS, PARTIAL_US, JOIN_US = (6.0, 1.0), (4.0, 1.0), 32, 1.7e-4, 0.08


def _unit_us(rows: np.ndarray) -> tuple:
    wide = rows > NARROW_ROWS
    return np.where(wide, WIDE_US[0], NARROW_US[0]), np.where(wide, WIDE_US[1], NARROW_US[1])


def choose_piece(runs: list, group: int, kv_heads: int, slots: int) -> int:
    """Into pieces of how many blocks the runs are cut: of some twenty sizes the one whose units, dealt to `slots`
    thread blocks the longest first, are done first. (Counting units alone, as many as there are slots, made
    pieces as long as the prompts where many short tails took the slots: 40 heads over 8, 30 sequences of 5
    prompts of 24,000 positions, 267 us a layer, now 49; 16 over 1, 8 of 2 prompts of 16,700: 19.5, now 14.4.)"""
    rows_of = np.array([len(members) * group for members, _, _ in runs], dtype=np.int64)
    sizes = np.array([c1 - c0 for _, c0, c1 in runs], dtype=np.int64)
    # (a run's rows: whole units and, where some are left, one more)
    rest = rows_of % UNIT_ROWS
    rows = np.concatenate([np.full_like(rest, UNIT_ROWS), rest])
    tiles = np.concatenate([rows_of // UNIT_ROWS, rest > 0])
    kept = tiles > 0
    rows, tiles, sizes = rows[kept], tiles[kept] * kv_heads, np.concatenate([sizes, sizes])[kept]
    starts, slopes = _unit_us(rows)
    rows = rows * tiles
    longest = int(sizes.max(initial=1))
    best, chosen, piece = math.inf, longest, max(1, int((sizes * tiles).sum() / (3 * slots)))
    while True:
        pieces = np.ceil(sizes / piece)
        costs = starts + slopes * np.ceil(sizes / pieces)
        counts = pieces * tiles
        least = float(costs.max())
        after = PARTIAL_US * float((pieces * rows).sum()) + JOIN_US * float(pieces.max())
        if max(least, float((costs * counts).sum()) / slots) + after < best:
            order = np.argsort(-costs)
            todo = np.repeat(costs[order], counts[order].astype(np.int64))
            done = np.zeros(slots)
            for i in range(0, len(todo), slots):
                some = todo[i:i + slots]
                done.sort()
                done[:len(some)] += some
            took = float(done.max()) + after
            if took < best:
                best, chosen = took, piece
        if piece >= longest or least >= best:
            return chosen
        piece = min(longest, piece + max(1, piece // 5))


class _Numbers(ctypes.Structure):
    """A plan's numbers as the launch takes them."""
    _fields_ = [(name, ctypes.c_int) for name in ("width", "unit_at", "unit_capacity", "member_at", "first_at",
                                                  "span_at", "partials", "sequences", "heads", "kv_heads")]


class SharedPlan:
    """Which pieces of the block lists are read for which sequences: int32 words on the device, and their
    layout. Right for every step until lengths pass `reach` (rounded up to whole blocks), fall below what is shared,
    or the sharing changes."""

    __slots__ = ("words", "sequences", "heads", "kv_heads", "units", "unit_at", "unit_capacity", "member_at",
                 "first_at", "span_at", "partials", "reach", "width", "saved", "numbers")

    @property
    def layout(self) -> tuple:
        """What a captured call keeps of a plan besides its words' address."""
        return (self.sequences, self.width, self.unit_capacity, self.member_at, self.first_at, self.partials)

    def on(self, words: torch.Tensor) -> "SharedPlan":
        """The same plan with its words at `words` (contiguous int32, on the device, at a multiple of 16 bytes)."""
        if words.dtype != torch.int32 or words.dim() != 1 or not words.is_contiguous() \
                or words.shape[0] < self.span_at + 2 * self.sequences or words.data_ptr() % 16:
            raise KernelError(f"SharedPlan: words must be contiguous int32 [{self.span_at + 2 * self.sequences} or more] "
                              f"at a multiple of 16 bytes, got {tuple(words.shape)} {words.dtype}")
        other = SharedPlan()
        for name in SharedPlan.__slots__:
            setattr(other, name, getattr(self, name))
        other.words = words
        return other


def _spread(counts: np.ndarray) -> tuple:
    """For `counts[i]` things each: the i of each thing, and its number among those of i."""
    of = np.repeat(np.arange(len(counts)), counts)
    return of, np.arange(len(of)) - (np.cumsum(counts) - counts)[of]


def _round_up(n: int, to: int) -> int:
    return -(-n // to) * to


def plan_shared(tables, lengths, heads: int, kv_heads: int, device=None, *, reach=None,
                slots: int | None = None, roomy: bool = False) -> SharedPlan:
    """The plan of `shared_decode_attention` for sequences whose block lists are `tables` (host integers
    [B, width], -1 for none) and which hold `lengths` positions (`reach`: how far they may grow before the
    plan is made again; default: as they are). `device` None leaves the words on the host (`words`: a
    numpy array); `roomy` rounds the layout's sizes up, so that plans of like shape have the same."""
    tables = np.asarray(tables)
    lengths = np.asarray(lengths, dtype=np.int64).reshape(-1)
    reach = lengths if reach is None else np.asarray(reach, dtype=np.int64).reshape(-1)
    if tables.ndim != 2 or tables.shape[0] != len(lengths) or len(reach) != len(lengths):
        raise KernelError(f"plan_shared: block lists {tables.shape} for {len(lengths)} lengths, {len(reach)} reaches")
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads or heads // kv_heads > MOST_GROUP:
        raise KernelError(f"plan_shared: {heads} heads over {kv_heads} (at most {MOST_GROUP} a KV head)")
    count, width = tables.shape
    if count and (lengths.min() < 0 or (reach < lengths).any() or reach.max() > width * CACHE_BLOCK):
        raise KernelError(f"plan_shared: lengths and reaches must lie in [0, {width * CACHE_BLOCK}], reach >= length")
    listed = np.arange(width)[None, :] < -(-lengths // CACHE_BLOCK)[:, None]
    if (tables[listed] < 0).any():
        raise KernelError("plan_shared: a sequence has positions without a block")
    group = heads // kv_heads
    runs = common_runs(tables, lengths, reach)
    piece = choose_piece(runs, group, kv_heads, slots or 2 * sm_count(device)) if runs else 1
    counted = np.array([len(members) for members, _, _ in runs], dtype=np.int64)
    ends = np.array([run[1:] for run in runs], dtype=np.int64).reshape(-1, 2)
    listing = np.array([b for members, _, _ in runs for b in members], dtype=np.int64)
    listed_at = np.cumsum(counted) - counted
    # the runs in even pieces, in the order of their positions
    sizes = ends[:, 1] - ends[:, 0]
    many = -(-sizes // piece)
    run, i = _spread(many)
    begins = ends[run, 0] + sizes[run] * i // many[run]
    columns = ends[run, 0] + sizes[run] * (i + 1) // many[run] - begins
    order = np.argsort(begins, kind="stable")
    run, begins, columns = run[order], begins[order], columns[order]
    # each piece's members; a sequence's partials lie in the order of its positions
    members = counted[run]
    pairs_at = np.cumsum(members) - members
    of, i = _spread(members)
    sequence = listing[listed_at[run[of]] + i]
    partial = np.empty_like(sequence)
    partial[np.argsort(sequence, kind="stable")] = np.arange(len(sequence))
    pairs = np.stack([sequence, partial], axis=1)
    first = np.concatenate([[0], np.cumsum(np.bincount(sequence, minlength=count))])
    # a piece's rows in units, those that take longest first
    rows = members * group
    of, i = _spread(-(-rows // UNIT_ROWS))
    r = i * UNIT_ROWS
    some = np.minimum(UNIT_ROWS, rows[of] - r)
    several = counted > 1
    units = np.stack([listing[listed_at[run[of]]], begins[of], columns[of], pairs_at[of] + r // group, r % group,
                      some, several[run[of]], np.zeros_like(of)], axis=1)
    start, slope = _unit_us(some)
    units = units[np.argsort(-(start + slope * columns[of]), kind="stable")]
    # the lengths that this holds for: what a sequence shares is filled, and its columns go no further
    spans = np.zeros((count, 2), dtype=np.int64)
    spans[:, 1] = -(-reach // CACHE_BLOCK) * CACHE_BLOCK
    shared = several[np.repeat(np.arange(len(counted)), counted)]
    np.maximum.at(spans[:, 0], listing[shared], np.repeat(ends[:, 1] * CACHE_BLOCK, counted)[shared])
    plan = SharedPlan()
    plan.sequences, plan.heads, plan.kv_heads, plan.width = count, heads, kv_heads, width
    plan.units, plan.reach = len(units), reach
    plan.unit_capacity = _round_up(len(units), 64) if roomy else len(units)
    members_room = _round_up(len(pairs), 256) if roomy else len(pairs)
    plan.partials = members_room                           # (a member is a partial)
    plan.unit_at = 8
    plan.member_at = plan.unit_at + UNIT_WORDS * plan.unit_capacity
    plan.first_at = plan.member_at + 2 * members_room
    plan.saved = int(((counted - 1) * sizes).sum())
    plan.span_at = plan.first_at + count + 1
    words = np.zeros(_round_up(plan.span_at + 2 * count, 4), dtype=np.int32)
    plan.numbers = _Numbers(*(getattr(plan, name) for name, _ in _Numbers._fields_))
    words[0], words[1] = len(units), count
    words[8:8 + UNIT_WORDS * len(units)] = units.reshape(-1)
    words[plan.member_at:plan.member_at + 2 * len(pairs)] = pairs.reshape(-1)
    words[plan.first_at:plan.first_at + count + 1] = first
    words[plan.span_at:plan.span_at + 2 * count] = spans.reshape(-1)
    plan.words = words if device is None else torch.from_numpy(words).to(device)
    return plan


def shared_decode_attention(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            seq_lens: torch.Tensor, block_table: torch.Tensor, plan: SharedPlan, heads: int,
                            kv_heads: int, head_dim: int, scale: float, *, settled: bool = False) -> torch.Tensor:
    """One query token per sequence over its cached keys and values, like `attention_decode` (bfloat16,
    head sizes 64 and 128, no window; `qkv`'s rows begin with the rotated queries, the newest key and value
    are in the cache), reading a block that `plan` found in several sequences' lists once for all of them.
    `plan`: `plan_shared` of these block lists. A sequence of length 0 gets zeros; one whose length the plan does not
    cover (past its reach, or below the blocks it shares) gets NaN, and so do those that the plan lets read those
    blocks through its list. `settled`: the plan's words, the lengths and the block lists were written before the kernel
    before this one on the stream began, as a step's inputs are; they are then read while that one still runs (else
    when it is done)."""
    q_shape, k_shape, device = qkv.shape, k_cache.shape, qkv.get_device()
    # (one expression for the calls that are right: a decode step outside a captured graph is bound by the
    # host's work; `_refuse` says what is wrong with the others)
    if not (qkv.dtype is torch.bfloat16 and k_cache.dtype is torch.bfloat16 and v_cache.dtype is torch.bfloat16
            and (head_dim == 128 or head_dim == 64) and 0 < kv_heads and heads % kv_heads == 0
            and heads <= MOST_GROUP * kv_heads and LEAST_SCALE <= scale <= 1 / LEAST_SCALE
            and len(q_shape) == 2 and q_shape[1] >= heads * head_dim
            and qkv.stride(1) == 1 and qkv.stride(0) % 2 == 0 and qkv.data_ptr() % 4 == 0
            and k_shape == v_cache.shape and len(k_shape) == 4 and k_cache.is_contiguous() and v_cache.is_contiguous()
            and k_shape[1] == kv_heads and k_shape[2] == CACHE_BLOCK and k_shape[3] == head_dim
            and seq_lens.dtype is torch.int32 and block_table.dtype is torch.int32
            and seq_lens.dim() == 1 and block_table.dim() == 2
            and seq_lens.shape[0] == q_shape[0] and block_table.shape[0] == q_shape[0]
            and block_table.shape[1] == plan.width and seq_lens.is_contiguous() and block_table.is_contiguous()
            and plan.sequences == q_shape[0] and plan.heads == heads and plan.kv_heads == kv_heads
            and plan.words.__class__ is torch.Tensor
            and device >= 0 and device == k_cache.get_device() == v_cache.get_device() == seq_lens.get_device()
            == block_table.get_device() == plan.words.get_device()):
        _refuse(qkv, k_cache, v_cache, seq_lens, block_table, plan, heads, kv_heads, head_dim, scale)
    sequences = q_shape[0]
    width = heads * head_dim
    out = torch.empty_like(qkv) if q_shape[1] == width and qkv.is_contiguous() else qkv.new_empty((sequences, width))
    if sequences == 0:
        return out
    part = qkv.new_empty(2 * plan.partials * heads * (head_dim + 2))          # (as many floats)
    call_on(device, "sakv_shared_attention", k_cache.data_ptr(), v_cache.data_ptr(), k_shape[0], qkv.data_ptr(),
            qkv.stride(0), seq_lens.data_ptr(), block_table.data_ptr(), plan.words.data_ptr(),
            ctypes.addressof(plan.numbers), out.data_ptr(), part.data_ptr(), head_dim, scale,
            bool(settled))
    if plan.unit_capacity:
        _lib.launches += 1          # the call launched the join too
    return out


def _refuse(qkv, k_cache, v_cache, seq_lens, block_table, plan, heads, kv_heads, head_dim, scale) -> None:
    """Says what is wrong with a call of `shared_decode_attention`."""
    if kv_heads <= 0 or not fast_path_takes(qkv.dtype, heads, kv_heads, head_dim):
        raise KernelError("shared_decode_attention: sizes not taken; use the plain kernel")
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] < heads * head_dim or qkv.stride(0) % 2 \
            or qkv.data_ptr() % 4:
        raise KernelError("shared_decode_attention: qkv must be [B, >= heads * head_dim], rows contiguous")
    for cache in (k_cache, v_cache):
        if cache.dim() != 4 or tuple(cache.shape[1:]) != (kv_heads, CACHE_BLOCK, head_dim) \
                or cache.shape != k_cache.shape or not cache.is_contiguous() or cache.dtype != torch.bfloat16:
            raise KernelError(f"shared_decode_attention: cache entries must be contiguous bf16 [blocks, {kv_heads}, "
                              f"{CACHE_BLOCK}, {head_dim}]")
    sequences = qkv.shape[0]
    for t, shape in ((seq_lens, (sequences,)), (block_table, (sequences, plan.width))):
        if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
            raise KernelError(f"shared_decode_attention: lengths and block lists must be contiguous int32, {shape}")
    if (plan.sequences, plan.heads, plan.kv_heads) != (sequences, heads, kv_heads):
        raise KernelError(f"shared_decode_attention: the plan is for {plan.sequences} sequences, {plan.heads} heads "
                          f"over {plan.kv_heads}")
    if not LEAST_SCALE <= scale <= 1 / LEAST_SCALE:
        raise KernelError(f"shared_decode_attention: scale must be a number from {LEAST_SCALE} to {1 / LEAST_SCALE}, "
                          f"got {scale}")
    if not isinstance(plan.words, torch.Tensor):
        raise KernelError("shared_decode_attention: the plan's words are on the host; `plan.on` takes them to the device")
    require_cuda(qkv, k_cache, v_cache, seq_lens, block_table, plan.words)
    raise KernelError("shared_decode_attention: tensors on different devices")
