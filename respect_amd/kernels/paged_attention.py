"""Attention of one new token per sequence over a paged KV cache.

No counterpart in the reference, which decodes one request over a contiguous buffer.
The HIP kernel (respect_amd/csrc/paged_attn.hip) splits every sequence by its own length
alone, so its result does not depend on the rest of the batch or on where its pages lie.
The cache's rows are bf16 or hold codes of 8 or 4 bits (``mx.MXRows``).  Where sequences of
a batch begin with the same rows, as forks of one prompt do, a ``SharedPrefix`` says so, and
those rows are read once for all of them.
"""
from __future__ import annotations

import operator

import numpy as np
import torch

from .. import _lib
from ._tensor import as_kernel_input, fits_32_bits
from .mx import MXRows, _pool_args


class SharedPrefix:
    """Which sequences of a batch begin alike: the first ``members[0]`` ones with the same
    ``keys[0]`` keys, the next ``members[1]`` with the same ``keys[1]``, and so on over the whole
    batch (0 keys, or one member: nothing is shared).  ``group``: query heads per kv head, up to 16.
    Made once for a batch and used by every layer and step, as long as the rows stay shared:
    sequences may grow, and any that has become shorter than its ``keys`` is taken by itself.  One
    that is as long again, but holds rows of its own there, needs a new plan.
    Whole steps of 64 keys are shared, the rest is left to the sequences (``prefix``)."""

    def __init__(self, members, keys, group: int, device="cuda"):
        m = np.array([operator.index(n) for n in members], dtype=np.int64)
        k = np.array([operator.index(n) for n in keys], dtype=np.int64)
        self.group = operator.index(group)
        if m.shape != k.shape or (m < 0).any() or (k < 0).any() or not 1 <= self.group <= 16:
            raise ValueError("SharedPrefix: members and keys must be equally many numbers >= 0, group 1 to 16")
        L, args = _lib.lib(), (m.ctypes.data, k.ctypes.data, len(m), self.group)
        count = L.rspx_shared_plan(*args, None, None)
        if count < 0:
            raise ValueError("SharedPrefix: at most 2^27 sequences and 2^31 - 1 keys")
        self.members, self.B, self.device = m.tolist(), sum(m.tolist()), torch.device(device)
        on_gpu = self.device.type == "cuda"
        if on_gpu and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("SharedPrefix: make the plan before a graph is captured")
        host = torch.empty(8 * count + self.B, dtype=torch.int32, pin_memory=on_gpu)
        at = host.data_ptr()
        L.rspx_shared_plan(*args, at + 32 * count, at)
        prefix = host[8 * count:].numpy()
        self.longest = int(prefix.max()) if self.B else 0
        first = np.minimum(m.cumsum() - m, max(self.B - 1, 0))
        self.groups = m, np.where(m > 0, prefix[first], 0).astype(np.int64) if self.B else 0 * k   # members, keys taken together
        flat = host.to(self.device)                # waited for: any stream may use the plan
        self.tiles, self.prefix = flat[:8 * count].view(count, 8), flat[8 * count:]


def paged_attn(q, kc, vc, table, lens, page: int, sm_scale=None, out=None, shared: SharedPrefix | None = None):
    """q [B, H, D], kc / vc [HK, slots, D] bf16 or ``MXRows`` of one format (one layer's pools:
    slots = pages * page), table [B, width] int32 page numbers, lens [B] int32 keys of each sequence, its new
    token's own among them -> [B, H, D] bf16.

    All on one GPU; table and lens are read there, so that a captured call follows them.
    A sequence of length 0 gets zeros; one whose length is negative or beyond its table, or
    that reads a page outside the pool, gets NaN.  ``page``: a power of two.  ``out``: written
    in place if given; no memory of the other tensors.  Scores as for ``prompt_attn``.

    ``shared``: which sequences begin alike.  The pages of the keys that a group shares are read
    from the table rows of sequences that have them all.  Probabilities of these keys are rounded to
    bf16, each by at most 2^-8 of itself (without ``shared`` by 2^-15), as in ``prompt_attn``, and an
    infinite value makes NaN where its probability is 0: the result is not that without ``shared`` bit
    for bit.  It depends on a sequence's own keys, length and shared keys, and not on who shares
    them.  The plan has to be kept as long as a graph that captured the call."""
    mx = isinstance(kc, MXRows)
    if out is None:
        if not mx and shared is None:
            name, y = "rspx_paged_attn", _lib.calls().paged_attn(q, kc, vc, table, lens, page, sm_scale)
        else:
            rows = (kc.codes, kc.scales, vc.codes, vc.scales, kc.bits) if mx and isinstance(vc, MXRows) and kc.format == vc.format \
                else (kc, None, vc, None, 16)
            plan = (None, None, 0, 0) if shared is None else (shared.prefix, shared.tiles, shared.longest, shared.group)
            name = "rspx_paged_attn_mx" if shared is None else "rspx_paged_attn_shared"
            y = _lib.calls().paged_attn_any(q, *rows, table, lens, page, sm_scale, *plan)
        if y is not None:
            return _lib.result(name, y)
    if mx != isinstance(vc, MXRows) or (mx and kc.format != vc.format):
        raise ValueError("paged_attn: the pools of K and V must be alike")
    if q.dim() != 3 or len(kc.shape) != 3 or kc.shape != vc.shape or kc.shape[2] != q.shape[2]:
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
    for name, t in () if mx else (("kc", kc), ("vc", vc)):       # a cache is never copied
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
    width, bits = table.shape[1], kc.bits if mx else 16
    if shared is not None:
        if shared.B != B or shared.longest > width * page:
            raise ValueError(f"paged_attn: the plan is one of {shared.B} sequences with up to {shared.longest} keys")
        if HK == 0 or H != HK * shared.group:
            raise ValueError(f"paged_attn: the plan is one of {shared.group} query heads per kv head")
        if shared.tiles.device != q.device:
            raise RuntimeError("paged_attn: the plan must be on the GPU of q")
    args = (q.data_ptr(), q.stride(0), q.stride(1), *_pool_args(kc), *_pool_args(vc), table.data_ptr(), table.stride(0),
            lens.data_ptr())
    plan = () if shared is None else (shared.prefix.data_ptr(), shared.tiles.data_ptr(), shared.tiles.shape[0], shared.longest)
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    with torch.cuda.device(q.device):
        # Of this call alone: torch hands it to the stream, or to the graph being captured.
        need = max(0, L.rspx_paged_attn_shared_workspace_bytes(B, H, D, page, width, 0 if shared is None else shared.longest, bits))
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        rest = (out.data_ptr(), out.stride(0), out.stride(1), B, H, HK, D, slots // page, page, width, scale)
        end = (ws.data_ptr() if need else None, need, _lib.stream_ptr(q.device))
        if shared is not None:
            name, rc = "rspx_paged_attn_shared", L.rspx_paged_attn_shared(*args, *plan, *rest, bits, *end)
        elif mx:
            name, rc = "rspx_paged_attn_mx", L.rspx_paged_attn_mx(*args, *rest, bits, *end)
        else:
            name, rc = "rspx_paged_attn", L.rspx_paged_attn(*args[:6], *args[9:12], *args[15:], *rest, *end)
    _lib.check(name, rc)
    return out
