"""Rows of a KV cache in the microscaled formats of 8 and 4 bits: written and read back.

No counterpart in the reference, whose cache is bf16.  32 consecutive elements of a row share
a power of two, a byte e that stands for 2^(e - 127): the smallest one (2^-117 at least) that
none of them outgrows.  An element is a number of 8 bits ("mxfp8": e4m3, up to 448) or of 4
("mxfp4": e2m1, up to 6; the first of two in the low half of a byte), rounded to nearest, ties
to even.  32 elements with an infinity or a NaN among them become NaN (e = 255).  Every value is
exact in bf16 (but that what rounds up to 2^128 is an infinity there), so what is read back is
what attention over the codes sees.  The HIP kernels are in
respect_amd/csrc/mx_rows.hip.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._tensor import as_kernel_input, fits_32_bits

BITS = {"mxfp8": 8, "mxfp4": 4}
GROUP = 32   # elements of a scale


class MXRows:
    """A pool of rows [HK, slots, D]: ``codes`` uint8 [HK, slots, D * bits / 8] (16-byte aligned
    rows) and ``scales`` uint8 [HK, slots, D / 32], of ``format`` "mxfp8" or "mxfp4"."""

    __slots__ = ("codes", "scales", "format", "bits", "shape", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, format: str):
        if format not in BITS:
            raise ValueError(f"MXRows: no format {format!r} (one of {', '.join(BITS)})")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("MXRows: codes and scales must be uint8")
        bits = BITS[format]
        if codes.dim() != 3 or scales.shape[:2] != codes.shape[:2] or codes.shape[2] % (4 * bits) or \
                scales.dim() != 3 or scales.shape[2] * 4 * bits != codes.shape[2]:
            raise ValueError(f"MXRows: {format} codes must be [HK, slots, D * {bits} / 8], scales [HK, slots, D / {GROUP}]")
        if codes.device != scales.device:
            raise ValueError("MXRows: codes and scales must be on one device")
        if codes.stride(2) != 1 or (scales.stride(2) != 1 and scales.shape[2] > 1) or codes.data_ptr() % 16 or \
                any(s % 16 for s in codes.stride()[:2]):
            raise ValueError("MXRows: rows must be contiguous, those of the codes 16-byte aligned")
        self.codes, self.scales, self.format, self.bits = codes, scales, format, bits
        self.shape = (*codes.shape[:2], codes.shape[2] * 8 // bits)
        self.device = codes.device

    @classmethod
    def empty(cls, HK: int, slots: int, D: int, format: str, device="cuda") -> "MXRows":
        """Rows of zeros."""
        if format not in BITS or D < GROUP or D % GROUP:
            raise ValueError(f"MXRows: head_dim a multiple of {GROUP}, format one of {', '.join(BITS)}")
        return cls(torch.zeros(HK, slots, D * BITS[format] // 8, dtype=torch.uint8, device=device),
                   torch.zeros(HK, slots, D // GROUP, dtype=torch.uint8, device=device), format)


def _pool_args(pool) -> tuple:
    """A pool's part of a C call: rows and scales, each with its head and slot strides."""
    if isinstance(pool, MXRows):
        c, s = pool.codes, pool.scales
        return c.data_ptr(), c.stride(0), c.stride(1), s.data_ptr(), s.stride(0), s.stride(1)
    return pool.data_ptr(), pool.stride(0), pool.stride(1), None, 0, 0


def _pools(what: str, kc, vc, slots: torch.Tensor) -> tuple[int, int, int, int]:
    """(HK, slots, D, bits) of a layer's pools; ``slots``: the rows' numbers."""
    if isinstance(kc, MXRows) != isinstance(vc, MXRows) or (isinstance(kc, MXRows) and kc.format != vc.format) or kc.shape != vc.shape:
        raise ValueError(f"{what}: the pools of K and V must be alike")
    if slots.dim() != 1:
        raise ValueError(f"{what}: slots must be [T]")
    if slots.dtype != torch.int32:
        raise TypeError(f"{what}: slots must be int32")
    HK, n, D = kc.shape
    fits_32_bits(what, HK, n, D, slots.shape[0])
    return HK, n, D, kc.bits if isinstance(kc, MXRows) else 16


def write_rows(k: torch.Tensor, v: torch.Tensor, kc: MXRows, vc: MXRows, slots: torch.Tensor) -> None:
    """k / v [T, HK, D] bf16 quantised into the rows ``slots`` [T] (device int32) of the pools kc /
    vc; a slot outside them is skipped, one named twice keeps parts of either row.  Can be captured."""
    if not isinstance(kc, MXRows) or not isinstance(vc, MXRows):
        raise TypeError("write_rows: the pools must be MXRows")
    y = _lib.calls().kv_write_mx(k, v, kc.codes, kc.scales, vc.codes, vc.scales, slots, kc.bits if kc.format == vc.format else 0)
    if y is not None:
        _lib.result("rspx_kv_write_mx", y)
        return
    HK, n, D, bits = _pools("write_rows", kc, vc, slots)
    T = slots.shape[0]
    if tuple(k.shape) != (T, HK, D) or v.shape != k.shape:
        raise ValueError(f"write_rows: k and v must be [{T}, {HK}, {D}]")
    k, v, slots = as_kernel_input(k, "k"), as_kernel_input(v, "v"), slots.contiguous()
    if any(t.device != kc.device for t in (k, v, slots, vc)):
        raise RuntimeError("write_rows: k, v and slots must be on the pools' GPU")
    with torch.cuda.device(kc.device):
        rc = _lib.lib().rspx_kv_write_mx(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(), T, n,
            *_pool_args(kc), *_pool_args(vc), HK, D, bits, _lib.stream_ptr(kc.device))
    _lib.check("rspx_kv_write_mx", rc)


def read_rows(kc, vc, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [T, HK, D] bf16: the rows ``slots`` [T] (device int32) of a layer's pools, MXRows or
    bf16 [HK, slots, D].  A slot outside them gives a row of NaN.  Can be captured."""
    if isinstance(kc, MXRows) and isinstance(vc, MXRows):
        y = _lib.calls().kv_read(kc.codes, kc.scales, vc.codes, vc.scales, slots, kc.bits if kc.format == vc.format else 0)
    else:
        y = _lib.calls().kv_read(kc, None, vc, None, slots, 16)
    if y is not None:
        return _lib.result("rspx_kv_read", y)
    HK, n, D, bits = _pools("read_rows", kc, vc, slots)
    if bits == 16:
        for name, t in (("kc", kc), ("vc", vc)):                     # a cache is never copied
            if as_kernel_input(t, name) is not t:
                raise ValueError(f"read_rows: {name} must have contiguous, 16-byte aligned rows")
    T = slots.shape[0]
    slots = slots.contiguous()
    if not kc.device.type == "cuda" or any(t.device != kc.device for t in (vc, slots)):
        raise RuntimeError("read_rows: the pools and slots must be on one GPU")
    k, v = (torch.empty((T, HK, D), dtype=torch.bfloat16, device=kc.device) for _ in range(2))
    with torch.cuda.device(kc.device):
        rc = _lib.lib().rspx_kv_read(
            *_pool_args(kc), *_pool_args(vc), slots.data_ptr(), T, n, k.data_ptr(), HK * D, D, v.data_ptr(), HK * D, D, HK, D,
            bits, _lib.stream_ptr(kc.device))
    _lib.check("rspx_kv_read", rc)
    return k, v
