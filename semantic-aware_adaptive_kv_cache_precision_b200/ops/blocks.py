"""Copies of cache blocks and of rows of per-sequence state (`csrc/copy_blocks.cu`). The reference's
pages belong to one sequence and are never copied (`src/core_kernels/kv_pages.cu:219-263`)."""

from __future__ import annotations

import array
import ctypes
import math
import operator

import torch

from ._lib import KernelError, call_on, require_cuda


class _Tensor(ctypes.Structure):
    _fields_ = [("source", ctypes.c_void_p), ("target", ctypes.c_void_p)] + [
        (name, ctypes.c_longlong) for name in ("source_entry", "target_entry", "block", "entries", "chunks",
                                               "chunk_bytes", "chunk_pitch")]


def _span(t: torch.Tensor) -> tuple:
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


def copy_blocks(tensors, src, dst, *, into=None, rows: int | None = None, axis: int = 1) -> None:
    """Block `src[n]` of every tensor becomes block `dst[n]`, all in one launch (up to 16 tensors and
    1,024 pairs; more take further launches).

    `tensors`: contiguous tensors whose dimension `axis` counts blocks: 1 for the cache's pools [entries,
    blocks, heads, 64, width], 0 for per-sequence state [slots, ...]. `src`, `dst`: block numbers on the
    host; a source may be copied to several targets, a target is named once. `into`: tensors of the same
    types and shapes but for the number of blocks that take the copies (default: `tensors` themselves; then
    no target may be a source). `rows` (axis 1, five dimensions): only the first `rows` positions of a
    block, the others stay as they are."""
    tensors = list(tensors)
    targets = tensors if into is None else list(into)
    if len(targets) != len(tensors):
        raise KernelError(f"copy_blocks: {len(tensors)} tensors into {len(targets)}")
    if axis != 0 and axis != 1:
        raise KernelError(f"copy_blocks: axis must be 0 or 1, got {axis}")
    if not tensors:
        return
    table = (_Tensor * len(tensors))()
    device = tensors[0].get_device()
    known, blocks, room, some = None, -1, -1, 0
    spans = []
    for t, u in zip(tensors, targets):
        shape = t.shape
        alike = (shape, t.dtype, None if u is t else u.shape)
        if alike != known:                 # (the keys' pool and the values' are mostly alike)
            known = alike
            geometry, blocks, room = _geometry(t, u, rows, axis, blocks, room)
        if not t.is_contiguous() or t.get_device() != device or u is not t and (
                not u.is_contiguous() or u.get_device() != device or u.dtype != t.dtype):
            raise KernelError(f"copy_blocks: {tuple(shape)} {t.dtype} into {tuple(u.shape)} {u.dtype}: contiguous "
                              "tensors of one type on one device")
        if t.numel() == 0:                 # (state of no size beside other state: nothing of it to copy)
            continue
        a, z = t.data_ptr(), u.data_ptr()
        table[some] = (a, z) + geometry
        some += 1
        spans.append((z, z + (geometry[1] or room * geometry[2]) * geometry[3]))
    src, dst = (ids if hasattr(ids, "__len__") else list(ids) for ids in (src, dst))     # (each is read twice, perhaps)
    try:
        source, target = array.array("i", src), array.array("i", dst)
    except (TypeError, OverflowError):                        # (numbers of other kinds, or past 32 bits)
        try:
            source, target = (array.array("q", map(operator.index, ids)) for ids in (src, dst))
        except (TypeError, OverflowError):
            raise KernelError("copy_blocks: sources and targets must be whole numbers") from None
        _check_numbers(source, target, blocks, room, into is None)
        source, target = array.array("i", source), array.array("i", target)
    count = len(source)
    if count != len(target):
        raise KernelError(f"copy_blocks: {count} sources, {len(target)} targets")
    if into is not None:
        if _overlap(spans, [_span(t) for t in tensors]):
            raise KernelError("copy_blocks: a target tensor overlaps another one")
    elif len(spans) > 1 and _overlap(spans):
        raise KernelError("copy_blocks: tensors overlap")
    if device < 0 or not some or not count:
        _check_numbers(source, target, blocks, room, into is None)
        require_cuda(*tensors)
        return
    try:
        call_on(device, "sakv_copy_blocks", table, some, source.buffer_info()[0], target.buffer_info()[0],
                count, blocks, room, into is None)
    except KernelError:
        _check_numbers(source, target, blocks, room, into is None)
        raise


def _check_numbers(source, target, blocks: int, room: int, within: bool) -> None:
    """Says what is wrong with the numbers of a copy, if anything is."""
    for ids, size, what in ((source, blocks, "sources"), (target, room, "targets")):
        if len(ids) and (min(ids) < 0 or max(ids) >= size):
            raise KernelError(f"copy_blocks: {what} must lie in [0, {size}), got [{min(ids)}, {max(ids)}]")
    if len(set(target)) != len(target):
        raise KernelError("copy_blocks: a target is named twice")
    if within and not set(target).isdisjoint(source):
        raise KernelError("copy_blocks: a target is a source too")


def _geometry(t, u, rows, axis, blocks, room) -> tuple:
    """((bytes from entry to entry here and there, bytes of a block, entries, chunks, bytes copied of a chunk,
    bytes from chunk to chunk), blocks here, blocks there) of tensors alike."""
    shape, there = t.shape, u.shape
    if len(shape) <= axis or len(shape) != len(there) or shape[:axis] != there[:axis] \
            or shape[axis + 1:] != there[axis + 1:]:
        raise KernelError(f"copy_blocks: {tuple(shape)} into {tuple(there)}: alike but for the number of blocks")
    if blocks >= 0 and (shape[axis], there[axis]) != (blocks, room):
        raise KernelError("copy_blocks: the tensors must have the same number of blocks")
    if rows is not None and (axis != 1 or len(shape) != 5 or not 0 < rows <= shape[3]):
        raise KernelError(f"copy_blocks: rows = {rows} of {tuple(shape)}")
    block = t.element_size() * math.prod(shape[axis + 1:])
    chunks, chunk, pitch = 1, block, block
    if rows is not None and rows < shape[3]:
        chunks, pitch = shape[2], block // max(1, shape[2])
        chunk = pitch // shape[3] * rows
    entry = (shape[1] * block, there[1] * block) if axis else (0, 0)       # (0: no entries)
    return entry + (block, shape[0] if axis else 1, chunks, chunk, pitch), shape[axis], there[axis]


def _overlap(spans: list, others: list = ()) -> bool:
    """Whether two of `spans` have bytes in common, or one of them with one of `others`."""
    ordered = sorted(spans)
    end = 0
    for a, z in ordered:
        if a < z:
            if a < end:
                return True
            end = z
    for a, z in others:
        for b, y in ordered:
            if a < z and b < y and a < y and b < z:
                return True
    return False
