"""Log-probabilities of given tokens under the output head, the vocabulary taken in pieces so that the
logits are never kept (`csrc/logprobs.cu`)."""

from __future__ import annotations

import ctypes

import torch

from . import gemm_wide
from ._lib import F32, KernelError, call, dtype_code, plain_function, ptr, require_cuda
from .linear import linear

#: logits that lie in memory at one time where a piece is a product of its own (fp32: 32 MB, a quarter of L2)
PIECE_ELEMENTS = 8 << 20


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
    bias_code = F32 if bias is None else dtype_code(bias.dtype)
    if not softcap >= 0.0 or softcap == float("inf"):
        raise KernelError(f"token_logprobs: softcap must be a number >= 0, got {softcap}")
    if any(t is not None and t.device != x.device for t in (head, targets, bias)):
        raise KernelError("token_logprobs: tensors on different devices")
    require_cuda(x, head, targets, bias)
    if rows == 1 or k == 1:                      # (strides that nothing depends on may be any number)
        x = x.as_strided((rows, k), (max(k, x.stride(0)) if rows > 1 else k, 1))
    form = (ptr(bias), bias_code, float(scale), float(softcap))
    device = x.get_device()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _token_logprobs(x, head, targets, bias, form)
    return _token_logprobs(x, head, targets, bias, form)


def _token_logprobs(x, head, targets, bias, form):
    rows, vocab, k = x.shape[0], head.shape[0], head.shape[1]
    logprob = x.new_empty(rows, dtype=torch.float32)
    lse, mine = x.new_empty(rows, dtype=torch.float32), x.new_empty(rows, dtype=torch.float32)
    if rows == 0:
        return logprob, lse
    if gemm_wide.takes(x, head) and _pairs() > 0:
        shape = (ctypes.c_int * 4)()
        if plain_function("sakv_logprob_shape")(rows, vocab, _pairs(), shape) != 0:
            raise KernelError(f"token_logprobs: {rows} rows over {vocab} tokens are too many")
        full, pieces, rest_pieces = shape[0] * 256, shape[2], 2 * shape[3]
        part = x.new_empty(2 * (pieces * full + rest_pieces * max(0, rows - full)), dtype=torch.float32)
        call("sakv_logprob_pieces", ptr(x), x.stride(0), ptr(head), rows, vocab, k, shape, ptr(targets),
             ptr(part), ptr(mine), *form)
    elif x.dtype == torch.float32:
        full, pieces, rest_pieces = rows, -(-vocab // plain_function("sakv_logprob_f32_columns")()), 0
        part = x.new_empty((pieces, rows, 2), dtype=torch.float32)
        call("sakv_logprob_f32", ptr(x), x.stride(0), ptr(head), rows, vocab, k, ptr(targets), ptr(part),
             ptr(mine), *form)
    else:
        columns = plain_function("sakv_logprob_fold_columns")()
        most = max(1, PIECE_ELEMENTS // columns)
        if rows > most:                # (the scratch of a piece stays as large as it is for these)
            parts = [_token_logprobs(x[i:i + most], head, targets[i:i + most], bias, form)
                     for i in range(0, rows, most)]
            return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
        piece = max(1, min(-(-vocab // columns), PIECE_ELEMENTS // (rows * columns))) * columns
        full, pieces, rest_pieces = rows, -(-vocab // columns), 0
        part = torch.empty((pieces, rows, 2), dtype=torch.float32, device=x.device)
        for first in range(0, vocab, piece):
            z = linear(x, head[first:first + piece], out_dtype=torch.float32)
            call("sakv_logprob_fold", ptr(z), z.stride(0), rows, z.shape[1], first, vocab, ptr(targets),
                 ptr(part[first // columns]), ptr(mine), *form)
    call("sakv_logprob_join", ptr(part), ptr(mine), ptr(targets), ptr(logprob), ptr(lse), rows, vocab, full, pieces,
         rest_pieces)
    return logprob, lse
