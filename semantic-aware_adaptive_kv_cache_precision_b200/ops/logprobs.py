"""Log-probabilities of given tokens under the output head, the vocabulary taken in pieces so that the
logits are never kept (`csrc/logprobs.cu`)."""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import F32, KernelError, call, dtype_code, plain_function, ptr, require_cuda, sm_count

#: numbers of the head that lie in memory a second time where it is copied to rows that TMA takes (512 MB), and its
#: rows among them (which bound what tiles of many rows of x leave)
PIECE_ELEMENTS = 256 << 20
PIECE_ROWS = 1 << 18
#: numbers of x that are split at one time in 32 bits (six bytes each: 384 MB)
SPLIT_ELEMENTS = 64 << 20
#: (maximum, sum) pairs that rows leave at one time, one a tile of the head (512 MB)
SPLIT_PAIRS = 64 << 20
#: the largest scale and cap: they and a cap's reciprocal stay 32-bit numbers, also times log2(e)
MOST_SHAPE = 1e30


_resident: dict = {}


def _pairs() -> int:
    """Pairs of SMs that hold the tensor-core kernel at one time (74 on a B200; 0: not here)."""
    device = torch.cuda.current_device()
    if device not in _resident:
        _resident[device] = int(plain_function("sakv_logprob_resident")())
    return _resident[device]


def token_logprobs(x: torch.Tensor, head: torch.Tensor, targets: torch.Tensor, bias: torch.Tensor | None = None,
                   *, scale: float = 1.0, softcap: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(log-probabilities, log of the sum of exponentials), each fp32 [T], of the tokens `targets` (int32
    [T]) under the logits `cap(scale * (x head^T + bias))`, cap(z) = softcap * tanh(z / softcap) where
    softcap > 0. `x` [T, K] and `head` [vocab, K] of one type, float32 or bfloat16; `bias` [vocab] float32 or
    bfloat16. A negative target asks for nothing and gets 0; one past the vocabulary gets NaN. A row with a
    logit that is NaN or +inf has NaN; logits of -inf count for nothing."""
    device, dtype = x.get_device(), x.dtype
    # (one expression for the calls that are right; `_refuse` says what is wrong with the others)
    if not (x.dim() == 2 and head.dim() == 2 and targets.dim() == 1 and dtype is head.dtype
            and (dtype is torch.bfloat16 or dtype is torch.float32) and x.stride(1) == 1 and head.is_contiguous()
            and 0 < x.shape[1] == head.shape[1] and head.shape[0] > 0
            and (x.stride(0) >= x.shape[1] or x.shape[0] <= 1)
            and targets.dtype is torch.int32 and targets.shape[0] == x.shape[0] and targets.is_contiguous()
            and (softcap == 0.0 or 1 / MOST_SHAPE <= softcap <= MOST_SHAPE) and -MOST_SHAPE <= scale <= MOST_SHAPE
            and device >= 0 and head.get_device() == device and targets.get_device() == device
            and (bias is None or bias.dim() == 1 and bias.shape[0] == head.shape[0] and bias.is_contiguous()
                 and bias.get_device() == device
                 and (bias.dtype is torch.float32 or bias.dtype is torch.bfloat16))):
        x = _refuse(x, head, targets, bias, scale, softcap)
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _token_logprobs(x, head, targets, bias, scale, softcap)
    return _token_logprobs(x, head, targets, bias, scale, softcap)


def _refuse(x, head, targets, bias, scale, softcap) -> torch.Tensor:
    """Says what is wrong with a call of `token_logprobs`, or gives x with strides that mean something (of one
    row, or one number a row, torch's may be any)."""
    if x.dim() != 2 or head.dim() != 2 or x.shape[1] != head.shape[1] or x.dtype != head.dtype \
            or head.shape[0] == 0 or x.shape[1] == 0:
        raise KernelError(f"token_logprobs: x {tuple(x.shape)} {x.dtype} does not fit the head {tuple(head.shape)} "
                          f"{head.dtype}")
    dtype_code(x.dtype)
    rows, vocab, k = x.shape[0], head.shape[0], head.shape[1]
    if x.stride(1) != 1 and k > 1 or rows > 1 and x.stride(0) < k or not head.is_contiguous():
        raise KernelError("token_logprobs: x rows and the head must be contiguous, x rows apart")
    if targets.dtype != torch.int32 or targets.shape != (rows,) or not targets.is_contiguous():
        raise KernelError(f"token_logprobs: targets must be contiguous int32 [{rows}]")
    if bias is not None and (bias.shape != (vocab,) or not bias.is_contiguous()):
        raise KernelError(f"token_logprobs: bias must be contiguous [{vocab}]")
    if bias is not None:
        dtype_code(bias.dtype)
    if not (softcap == 0.0 or 1 / MOST_SHAPE <= softcap <= MOST_SHAPE) or not -MOST_SHAPE <= scale <= MOST_SHAPE:
        raise KernelError(f"token_logprobs: softcap must be 0 or a number from {1 / MOST_SHAPE} to {MOST_SHAPE}, scale one "
                          f"of at most {MOST_SHAPE}, got {softcap} and {scale}")
    if any(t is not None and t.device != x.device for t in (head, targets, bias)):
        raise KernelError("token_logprobs: tensors on different devices")
    require_cuda(x, head, targets, bias)
    return x.as_strided((rows, k), (max(k, x.stride(0)) if rows > 1 else k, 1))


_shapes: dict = {}


def _shape(rows: int, vocab: int, k: int):
    """How the tensor-core kernel cuts so many rows and tokens on this device: (the numbers the launch takes, floats
    of scratch)."""
    pairs = _pairs()
    hit = _shapes.get((rows, vocab, k, pairs))
    if hit is None:
        shape = (ctypes.c_int * 4)()
        if plain_function("sakv_logprob_shape")(rows, vocab, k, pairs, shape) != 0:
            raise KernelError(f"token_logprobs: {rows} rows over {vocab} tokens are too many")
        full = shape[0] * 256
        if len(_shapes) >= 256:
            _shapes.clear()
        hit = _shapes[rows, vocab, k, pairs] = (shape, 2 * (shape[2] * full + 2 * shape[3] * max(0, rows - full)))
    return hit


_heights: dict = {}


def _split_rows(vocab: int) -> int:
    """Rows of the head in a tile of the 32-bit tensor-core kernel on this device."""
    sms = sm_count()
    hit = _heights.get((vocab, sms))
    if hit is None:
        if len(_heights) >= 256:
            _heights.clear()
        hit = _heights[vocab, sms] = plain_function("sakv_logprob_split_rows")(vocab, sms)
    return hit


def _in_pieces(x, head, targets, bias, scale, softcap, most: int):
    """So many rows at a time."""
    parts = [_token_logprobs(x[i:i + most], head, targets[i:i + most], bias, scale, softcap)
             for i in range(0, x.shape[0], most)]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def _token_logprobs(x, head, targets, bias, scale, softcap, found=None):
    """`found` (rows of 16 bits that TMA takes, as many as one launch may have): gets the targets' logits."""
    rows, k = x.shape
    vocab, stride = head.shape[0], x.stride(0)
    logprob, lse = x.new_empty(rows, dtype=torch.float32), x.new_empty(rows, dtype=torch.float32)
    if rows == 0:
        return logprob, lse
    if rows == 1:
        stride = k
    at, head_at = x.data_ptr(), head.data_ptr()
    bias_at, bias_code = (None, F32) if bias is None else (bias.data_ptr(), dtype_code(bias.dtype))
    if x.dtype is torch.bfloat16 and k % 8 == 0 and stride % 8 == 0 and (at | head_at) % 16 == 0 and _pairs() > 0:
        shape, floats = _shape(rows, vocab, k)
        if floats > 2 * SPLIT_PAIRS and rows > 256 and found is None:
            # (whole tiles of 256 rows; the heads' tiles of fewer rows may be lower ones, so a piece is looked at again)
            return _in_pieces(x, head, targets, bias, scale, softcap,
                              max(256, min(rows - 1, rows * 2 * SPLIT_PAIRS // floats) // 256 * 256))
        part = x.new_empty(floats + rows, dtype=torch.float32)
        scratch = part.data_ptr()
        call("sakv_logprob_pieces", at, stride, head_at, rows, vocab, k, shape, targets.data_ptr(), scratch,
             scratch + 4 * floats, bias_at, bias_code, scale, softcap, logprob.data_ptr(), lse.data_ptr())
        _lib.launches += 1          # the call launched the join too
        if found is not None:
            found.copy_(part[floats:])
    elif x.dtype is torch.float32 and k % 4 == 0 and head_at % 16 == 0:
        padded, tile = -(-k // 8) * 8, _split_rows(vocab)
        most = max(1, min(SPLIT_ELEMENTS // padded, SPLIT_PAIRS // -(-vocab // tile)))
        if rows > most:
            return _in_pieces(x, head, targets, bias, scale, softcap, most)
        halves = 3 * plain_function("sakv_logprob_split_tokens")(rows) * padded // 2
        floats = halves + 2 * rows * -(-vocab // tile)
        part = x.new_empty(floats + rows, dtype=torch.float32)       # the split rows, the partials, the targets' logits
        scratch = part.data_ptr()
        call("sakv_logprob_split", at, stride, head_at, rows, vocab, k, tile, targets.data_ptr(), scratch + 4 * halves,
             scratch + 4 * floats, scratch, bias_at, bias_code, scale, softcap, logprob.data_ptr(), lse.data_ptr())
        _lib.launches += 2          # the call launched the split of x and the join too
    elif x.dtype is torch.float32:
        pieces = -(-vocab // plain_function("sakv_logprob_f32_columns")())
        most = max(1, SPLIT_PAIRS // pieces)
        if rows > most:
            return _in_pieces(x, head, targets, bias, scale, softcap, most)
        floats = 2 * rows * pieces
        part = x.new_empty(floats + rows, dtype=torch.float32)
        scratch = part.data_ptr()
        call("sakv_logprob_f32", at, stride, head_at, rows, vocab, k, targets.data_ptr(), scratch,
             scratch + 4 * floats, bias_at, bias_code, scale, softcap, logprob.data_ptr(), lse.data_ptr())
        _lib.launches += 1
    else:                           # bfloat16 rows that TMA cannot take
        return _copied(x, head, targets, bias, scale, softcap)
    return logprob, lse


def _copied(x, head, targets, bias, scale, softcap):
    """bfloat16 rows whose size is no multiple of 8, or that do not begin at multiples of 16 bytes: from copies that are
    and do, of x and, where it takes one, of the head, a piece of it at a time. (A piece's partial is its log of the sum of
    exponentials: it stands for one maximum beside a sum of 1.) 64 rows of 1,535 over 151,936: 267 us, of which the copy
    takes 177; 2,047 rows 745."""
    if _pairs() <= 0:
        raise KernelError("token_logprobs: no pair of this device's SMs holds the kernel")
    rows, k = x.shape
    vocab, padded = head.shape[0], -(-k // 8) * 8
    if k == padded and head.data_ptr() % 16 == 0:
        return _token_logprobs(_padded(x, x.new_empty((rows, k))), head, targets, bias, scale, softcap)
    piece = min(vocab, max(1, min(PIECE_ELEMENTS // padded, PIECE_ROWS)))
    most = max(256, SPLIT_PAIRS // -(-piece // 192) // 256 * 256)        # (tiles of the head have 192 rows at least)
    if rows > most:
        return _in_pieces(x, head, targets, bias, scale, softcap, most)
    x, room = _padded(x, x.new_empty((rows, padded))), x.new_empty((piece, padded))
    if piece == vocab:
        return _token_logprobs(x, _padded(head, room), targets, bias, scale, softcap)
    pieces = -(-vocab // piece)
    part = x.new_empty((pieces, rows, 2), dtype=torch.float32)
    mine, found = x.new_zeros(rows, dtype=torch.float32), x.new_empty(rows, dtype=torch.float32)
    for i, first in enumerate(range(0, vocab, piece)):
        n = min(piece, vocab - first)
        here = (targets >= first) & (targets < first + n)
        _, lse = _token_logprobs(x, _padded(head[first:first + n], room[:n]), torch.where(here, targets - first, -1),
                                 None if bias is None else bias[first:first + n], scale, softcap, found)
        part[i, :, 0] = lse
        part[i, :, 1] = lse != -float("inf")
        mine = torch.where(here, found, mine)
    logprob, lse = x.new_empty(rows, dtype=torch.float32), x.new_empty(rows, dtype=torch.float32)
    call("sakv_logprob_join", ptr(part), ptr(mine), ptr(targets), ptr(logprob), ptr(lse), rows, vocab, pieces)
    return logprob, lse


def _padded(rows: torch.Tensor, into: torch.Tensor) -> torch.Tensor:
    """`rows` at the front of the rows of `into`, zeros behind them."""
    count, k = rows.shape
    call("sakv_logprob_pad", rows.data_ptr(), k if count == 1 else rows.stride(0), count, k, into.shape[1], into.data_ptr())
    return into
