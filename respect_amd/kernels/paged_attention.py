"""Attention of one new token per sequence over a paged KV cache.

No counterpart in the reference, which decodes one request over a contiguous buffer.
The HIP kernel (respect_amd/csrc/paged_attn.hip) splits every sequence by its own length
alone, so its result does not depend on the rest of the batch or on where its pages lie.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._tensor import as_kernel_input, fits_32_bits


def paged_attn(q, kc, vc, table, lens, page: int, sm_scale=None, out=None):
    """q [B, H, D], kc / vc [HK, slots, D] bf16 (one layer's pools: slots = pages * page),
    table [B, width] int32 page numbers, lens [B] int32 keys of each sequence, its new
    token's own among them -> [B, H, D] bf16.

    All on one GPU; table and lens are read there, so that a captured call follows them.
    A sequence of length 0 gets zeros; one whose length is negative or beyond its table, or
    that reads a page outside the pool, gets NaN.  ``page``: a power of two.  ``out``: written
    in place if given; no memory of the other tensors.  Scores as for ``prompt_attn``."""
    if out is None:
        y = _lib.calls().paged_attn(q, kc, vc, table, lens, page, sm_scale)
        if y is not None:
            return _lib.result("rspx_paged_attn", y)
    if q.dim() != 3 or kc.dim() != 3 or kc.shape != vc.shape or kc.shape[2] != q.shape[2]:
        raise ValueError("paged_attn: q must be [B, H, D], kc and vc [HK, slots, D]")
    B, H, D = q.shape
    HK, slots, _ = kc.shape
    if page < 1 or slots % page:
        raise ValueError(f"paged_attn: {slots} slots are no whole pages of {page}")
    if table.dim() != 2 or table.shape[0] != B or tuple(lens.shape) != (B,):
        raise ValueError(f"paged_attn: table must be [{B}, width] and lens [{B}]")
    fits_32_bits("paged_attn", B, H, HK, slots, page, table.shape[1])
    if table.dtype != torch.int32 or lens.dtype != torch.int32:
        raise TypeError("paged_attn: table and lens must be int32")
    for name, t in (("kc", kc), ("vc", vc)):                     # a cache is never copied
        if as_kernel_input(t, name) is not t:
            raise ValueError(f"paged_attn: {name} must have contiguous, 16-byte aligned rows")
    q = as_kernel_input(q, "q")
    if table.shape[1] > 1 and table.stride(1) != 1:
        table = table.contiguous()
    lens = lens.contiguous()
    if any(t.device != q.device for t in (kc, vc, table, lens)):
        raise RuntimeError("paged_attn: all tensors must be on one GPU")
    if out is None:
        out = torch.empty((B, H, D), dtype=torch.bfloat16, device=q.device)
    elif out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != q.device or out.stride(2) != 1:
        raise ValueError(f"paged_attn: out must be a bf16 {tuple(q.shape)} tensor with contiguous rows, on the GPU of q")
    L = _lib.lib()
    width = table.shape[1]
    with torch.cuda.device(q.device):
        # Of this call alone: torch hands it to the stream, or to the graph being captured.
        need = max(0, L.rspx_paged_attn_workspace_bytes(B, H, D, page, width))
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        rc = L.rspx_paged_attn(
            q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), kc.stride(0), kc.stride(1), vc.data_ptr(),
            vc.stride(0), vc.stride(1), table.data_ptr(), table.stride(0), lens.data_ptr(), out.data_ptr(),
            out.stride(0), out.stride(1), B, H, HK, D, slots // page, page, width,
            D ** -0.5 if sm_scale is None else float(sm_scale), ws.data_ptr() if need else None, need,
            _lib.stream_ptr(q.device))
    _lib.check("rspx_paged_attn", rc)
    return out
