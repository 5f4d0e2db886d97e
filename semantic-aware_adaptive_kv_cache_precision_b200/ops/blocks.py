"""Copies of cache blocks and of rows of per-sequence state (`csrc/copy_blocks.cu`). The reference's
pages belong to one sequence and are never copied (`src/core_kernels/kv_pages.cu:219-263`)."""

from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import KernelError, call, on_device, require_cuda


class _Tensor(ctypes.Structure):
    _fields_ = [("source", ctypes.c_void_p), ("target", ctypes.c_void_p)] + [
        (name, ctypes.c_longlong) for name in ("source_entry", "target_entry", "block", "entries", "chunks",
                                               "chunk_bytes", "chunk_pitch")]


def _span(t: torch.Tensor) -> tuple:
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


def _ids(ids, size: int, what: str) -> list:
    ids = [int(i) for i in ids]
    if ids and (min(ids) < 0 or max(ids) >= size):
        raise KernelError(f"copy_blocks: {what} must lie in [0, {size}), got [{min(ids)}, {max(ids)}]")
    return ids


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
    if axis not in (0, 1):
        raise KernelError(f"copy_blocks: axis must be 0 or 1, got {axis}")
    if not tensors:
        return
    table = (_Tensor * len(tensors))()
    blocks, room = tensors[0].shape[axis] if tensors[0].dim() > axis else 0, None
    for i, (t, u) in enumerate(zip(tensors, targets)):
        if t.dim() <= axis or t.dim() != u.dim() or t.dtype != u.dtype or t.device != u.device \
                or t.device != tensors[0].device or not t.is_contiguous() or not u.is_contiguous() \
                or t.shape[:axis] != u.shape[:axis] or t.shape[axis + 1:] != u.shape[axis + 1:]:
            raise KernelError(f"copy_blocks: {tuple(t.shape)} {t.dtype} into {tuple(u.shape)} {u.dtype}: contiguous "
                              "tensors on one device, alike but for the number of blocks")
        if t.shape[axis] != blocks or (room is not None and u.shape[axis] != room):
            raise KernelError("copy_blocks: the tensors must have the same number of blocks")
        room = u.shape[axis]
        if rows is not None and (axis != 1 or t.dim() != 5 or not 0 < rows <= t.shape[3]):
            raise KernelError(f"copy_blocks: rows = {rows} of {tuple(t.shape)}")
        size = t.element_size()
        entry = t.numel() // t.shape[0] * size if axis else 0       # (0 where there are no entries)
        block = size
        for n in t.shape[axis + 1:]:
            block *= n
        chunks, chunk, pitch = 1, block, block
        if rows is not None and rows < t.shape[3]:
            chunks, pitch = t.shape[2], t.shape[3] * t.shape[4] * size
            chunk = pitch // t.shape[3] * rows
        table[i] = _Tensor(t.data_ptr(), u.data_ptr(), entry, u.shape[1] * block if axis else 0, block,
                           t.shape[0] if axis else 1, chunks, chunk, pitch)
    src, dst = _ids(src, blocks, "sources"), _ids(dst, room, "targets")
    if len(src) != len(dst):
        raise KernelError(f"copy_blocks: {len(src)} sources, {len(dst)} targets")
    if len(set(dst)) != len(dst):
        raise KernelError("copy_blocks: a target is named twice")
    if into is None:
        if not set(dst).isdisjoint(src):
            raise KernelError("copy_blocks: a target is a source too")
        if _overlap([_span(t) for t in tensors]):
            raise KernelError("copy_blocks: tensors overlap")
    elif _overlap([_span(t) for t in targets], [_span(t) for t in tensors]):
        raise KernelError("copy_blocks: a target tensor overlaps another one")
    require_cuda(*tensors, *targets)
    if not src or any(t.numel() == 0 for t in tensors):
        return
    pairs = np.empty((len(src), 2), dtype=np.int32)
    pairs[:, 0], pairs[:, 1] = src, dst
    with on_device(tensors[0]):
        call("sakv_copy_blocks", ctypes.addressof(table), len(tensors), pairs.ctypes.data, len(src))


def _overlap(spans: list, others: list = ()) -> bool:
    """Whether two of `spans` have bytes in common, or one of them with one of `others`."""
    ordered = sorted(s for s in spans if s[0] < s[1])
    if any(a[1] > b[0] for a, b in zip(ordered, ordered[1:])):
        return True
    return any(a[0] < b[1] and b[0] < a[1] for a in ordered for b in others if b[0] < b[1])
