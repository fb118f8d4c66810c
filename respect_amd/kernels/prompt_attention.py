"""Causal attention over whole prompts of different lengths, packed one after the other.

No counterpart in the reference, which prefills one request with stock SDPA.  The
tokens of all prompts lie in one [T, heads, D] tensor; a ``PackedPrompts`` says which rows
belong together, made once for a batch and used by every layer.  The HIP kernel
(respect_amd/csrc/prompt_attn.hip) computes a row from its own sequence's keys in a fixed
order: its bits do not depend on what else is packed beside it.
"""
from __future__ import annotations

import operator

import numpy as np
import torch

from .. import _lib
from ._tensor import as_kernel_input, fits_32_bits

TILE_ROWS = (32, 64, 128)   # what rspx_prompt_attn_tile_rows gives


class PackedPrompts:
    """The layout of a packed batch.  ``rows[s]``: tokens of sequence s in q; ``keys[s]``
    (default: the same): its tokens in k and v.  Causal from the end: the last row of a
    sequence sees all its keys, the row before it one fewer; with keys > rows the first
    keys are earlier ones (a cached beginning), with keys < rows the first rows see nothing
    and get zeros."""

    def __init__(self, rows, keys=None, device="cuda"):
        r = np.array([operator.index(n) for n in rows], dtype=np.int64)
        k = r if keys is None else np.array([operator.index(n) for n in keys], dtype=np.int64)
        if r.shape != k.shape or (r < 0).any() or (k < 0).any():
            raise ValueError("PackedPrompts: rows and keys must be equally many lengths >= 0")
        self.rows, self.keys = r.tolist(), k.tolist()
        self.Tq, self.Tk = sum(self.rows), sum(self.keys)
        self.device = torch.device(device)
        L, args = _lib.lib(), (r.ctypes.data, k.ctypes.data, len(r))
        count = [L.rspx_prompt_attn_tiles(*args, size, None) for size in TILE_ROWS]
        if min(count) < 0:
            raise ValueError("PackedPrompts: at most 2^31 - 1 tokens")
        on_gpu = self.device.type == "cuda"
        if on_gpu and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PackedPrompts: make the plan before a graph is captured")
        host = torch.empty((sum(count), 4), dtype=torch.int32, pin_memory=on_gpu)
        at = host.data_ptr()
        for size, n in zip(TILE_ROWS, count):
            if n:
                L.rspx_prompt_attn_tiles(*args, size, at)
            at += 16 * n
        self._lists = host.to(self.device).split(count)   # waited for: any stream may use the plan

    def tiles(self, H: int, HK: int) -> torch.Tensor:
        """Device int32 [n, 4]: the tiles rspx_prompt_attn takes for these heads."""
        return self._lists[TILE_ROWS.index(_lib.lib().rspx_prompt_attn_tile_rows(H, HK))]


def prompt_attn(q, k, v, plan: PackedPrompts, sm_scale=None, out=None):
    """q [Tq, H, D], k / v [Tk, HK, D] bf16, packed as ``plan`` says -> [Tq, H, D] bf16.
    ``sm_scale``: default D ** -0.5.  ``out``: written in place if given (any strides with
    D contiguous, multiples of 8 elements; no memory of k's or v's, of q's only as q itself).  Scores up to 5e8 in
    magnitude: past that the softmax's exponents lose their fp32 range and NaN may come."""
    if out is None and isinstance(plan, PackedPrompts):
        y = _lib.calls().prompt_attn(q, k, v, plan.Tq, plan.Tk, *plan._lists, sm_scale)
        if y is not None:
            return _lib.result("rspx_prompt_attn", y)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise ValueError("prompt_attn: q must be [Tq, H, D], k and v [Tk, HK, D]")
    T, H, D = q.shape
    Tk, HK, _ = k.shape
    if T != plan.Tq or Tk != plan.Tk:
        raise ValueError(f"prompt_attn: the plan packs {plan.Tq} rows and {plan.Tk} keys, not {T} and {Tk}")
    fits_32_bits("prompt_attn", H, HK)
    if HK == 0 or H % HK:
        raise ValueError(f"prompt_attn: {H} heads over {HK} kv heads")
    q, k, v = (as_kernel_input(t, n) for t, n in ((q, "q"), (k, "k"), (v, "v")))
    tiles = plan.tiles(H, HK)
    if not q.device == k.device == v.device == tiles.device:
        raise RuntimeError("prompt_attn: q, k, v and the plan must be on one GPU")
    if out is None:
        out = torch.empty((T, H, D), dtype=torch.bfloat16, device=q.device)
    elif out.shape != q.shape or as_kernel_input(out, "out") is not out or out.device != q.device:
        raise ValueError(f"prompt_attn: out must be a bf16 {tuple(q.shape)} tensor with aligned rows, on the GPU of q")
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    with torch.cuda.device(q.device):
        rc = _lib.lib().rspx_prompt_attn(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
            v.stride(1), tiles.data_ptr(), tiles.shape[0], out.data_ptr(), out.stride(0), out.stride(1), H, HK, T, Tk, D,
            scale, _lib.stream_ptr(q.device))
    _lib.check("rspx_prompt_attn", rc)
    return out
