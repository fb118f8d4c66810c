"""Log probabilities of given tokens, entropy and the best alternatives, beside the greedy
choice of ``acceptance`` and over the same scores.  No counterpart in the reference."""
from __future__ import annotations

import operator

import torch

from .. import _lib
from ..kernels._tensor import fits_32_bits

MAX_TOP = 64   # alternatives rspx_token_logprobs gives at most


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, offset: int = 0, size: int = 0):
    """logits [M, V] fp32, tokens [M] int64, on one GPU -> (given [M], entropy [M], values
    [M, n], ids [M, n] int64), n = min(top, V): log p of each row's token, the row's entropy in
    nats, and its n largest scores' log p and columns, best first, ties to the lowest column.

    Columns [offset, offset + size) count as -inf, as for ``greedy_token``.  A token outside
    the vocabulary gets NaN; a row with NaN or +inf scores has NaN results, NaN first among
    the ids; a row with nothing left has -inf and entropy 0.  ``top`` <= 64."""
    y = _lib.calls().token_logprobs(logits, tokens, top, offset, size)
    if y is not None:
        return _lib.result("rspx_token_logprobs", y)
    if logits.dtype != torch.float32 or not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
        raise TypeError("token_logprobs: fp32 [M, V] GPU logits with contiguous rows are required")
    M, V = logits.shape
    if tokens.dtype != torch.int64 or tuple(tokens.shape) != (M,) or tokens.device != logits.device:
        raise TypeError(f"token_logprobs: tokens must be int64 [{M}] on the GPU of the logits")
    if V == 0 or not 0 <= top <= MAX_TOP:
        raise ValueError(f"token_logprobs: V {V}, top {top} (0 to {MAX_TOP})")
    fits_32_bits("token_logprobs", M, V)
    if logits.stride(0) < V:   # rows that overlap
        logits = logits.clone(memory_format=torch.contiguous_format)
    # Past the vocabulary or below 0 one number is as good as another: 32 bits hold these.
    offset, size = (min(max(operator.index(x), -1), V) for x in (offset, size))
    tokens = tokens.contiguous()
    dev, n = logits.device, min(top, V)
    given, entropy = torch.empty((2, M), dtype=torch.float32, device=dev)
    values = torch.empty((M, n), dtype=torch.float32, device=dev)
    ids = torch.empty((M, n), dtype=torch.int64, device=dev)
    L = _lib.lib()
    with torch.cuda.device(dev):
        # Of this call alone: torch hands it to the stream, or to the graph being captured.
        ws = torch.empty(L.rspx_token_logprobs_workspace_bytes(M, V, n), dtype=torch.uint8, device=dev)
        rc = L.rspx_token_logprobs(logits.data_ptr(), logits.stride(0), M, V, offset, size, tokens.data_ptr(),
                                   n, given.data_ptr(), entropy.data_ptr(), values.data_ptr(), ids.data_ptr(),
                                   ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
    _lib.check("rspx_token_logprobs", rc)
    return given, entropy, values, ids
