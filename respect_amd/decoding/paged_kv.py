"""KV cache of many sequences in pages: taken, shared, copied, compacted and given back.

No counterpart in the reference, whose buffer holds one request (kv_buffer.py here).
Per layer one bf16 pool [HK, pages * page, D] for K and one for V; row j of a sequence is
pool row ``table[j // page] * page + j % page``.  Who holds which page is kept on the
host (rspx_pages_*: pages are counted, so that forks share the full ones); the rows move on
the GPU, all layers and sequences in one launch (rspx_kv_move).  ``paged_attn`` reads the
pools through ``tables``.
"""
from __future__ import annotations

import ctypes
import operator

import numpy as np
import torch

from .. import _lib
from ..kernels._tensor import as_kernel_input, fits_32_bits


def _p(a: np.ndarray) -> int:
    return a.ctypes.data


def _whole(numbers) -> np.ndarray:
    """int64 of an iterable of whole numbers (``TypeError`` for any other: none is cut to one)."""
    return np.array([operator.index(x) for x in numbers], dtype=np.int64)


class PageTable:
    """Who holds which page, without the pools: the host half of ``PagedKVCache``.  A refused
    call (``ValueError``: no such sequence, one named twice, a bad count; ``TypeError``: not a
    whole number; ``RuntimeError``: too few pages or sequences) changes nothing."""

    def __init__(self, pages: int, page: int, sequences: int):
        self._lib = _lib.lib()
        self.handle = None
        if all(0 < operator.index(n) < 1 << 31 for n in (pages, page, sequences)):   # what 32 bits hold
            self.handle = self._lib.rspx_pages_new(pages, page, sequences)
        if not self.handle:
            raise ValueError("PagedKVCache: pages and sequences >= 1, page a power of two, pages * page below 2^31")

    def __del__(self):
        if getattr(self, "handle", None):
            self._lib.rspx_pages_delete(self.handle)
            self.handle = None

    def _call(self, what: str, *args) -> None:
        rc = getattr(self._lib, "rspx_pages_" + what)(self.handle, *args)
        if rc < 0:
            self.refuse(what, rc)

    @staticmethod
    def refuse(what: str, rc: int) -> None:
        """Raise what status ``rc`` of a bookkeeping call stands for."""
        if rc == -1:
            raise ValueError(f"PagedKVCache.{what}: no such sequence, one named twice, or a bad count, row or path")
        raise RuntimeError(f"PagedKVCache.{what}: {_lib.strerror(rc)} ({rc})")

    @staticmethod
    def _ids(seqs) -> np.ndarray:
        ids = _whole(seqs)
        if ids.size and (ids.min() < 0 or ids.max() >= 1 << 31):
            raise ValueError("PagedKVCache: no such sequence")
        return ids.astype(np.int32)

    @staticmethod
    def _counts(n, many: int) -> np.ndarray:
        """One number for each of ``many``, or that many of them."""
        if not np.iterable(n):
            return np.full(many, operator.index(n), np.int64)
        c = _whole(n)
        if len(c) != many:
            raise ValueError(f"PagedKVCache: {many} counts are needed")
        return c

    @property
    def available(self) -> int:
        return self._lib.rspx_pages_available(self.handle)

    def length(self, seq: int) -> int:
        n = self._lib.rspx_pages_length(self.handle, seq) if 0 <= seq < 1 << 31 else -1
        if n < 0:
            raise ValueError("PagedKVCache: no such sequence")
        return n

    def add(self, lengths) -> list[int]:
        n = _whole(lengths)
        ids = np.empty(len(n), np.int32)
        self._call("add", _p(n), len(n), _p(ids))
        return ids.tolist()

    def extend(self, seqs, n) -> None:
        ids = self._ids(seqs)
        self._call("extend", _p(ids), len(ids), _p(self._counts(n, len(ids))))

    def fork(self, seqs, copies: int) -> list[int]:
        ids = self._ids(seqs)
        copies = operator.index(copies)
        if not 0 <= copies < 1 << 31:
            raise ValueError("PagedKVCache: counts must be >= 0")
        if len(ids) * copies >= 1 << 24:
            self.refuse("fork", -6)
        out = np.empty(len(ids) * copies, np.int32)
        self._call("fork", _p(ids), len(ids), copies, _p(out))
        return out.tolist()

    def compact(self, seqs, starts, paths) -> None:
        ids = self._ids(seqs)
        paths = [_whole(p) for p in paths]
        if len(paths) != len(ids):
            raise ValueError("PagedKVCache: one path per sequence")
        flat = np.concatenate(paths) if paths else np.zeros(0, np.int64)
        ends = np.cumsum([len(p) for p in paths], dtype=np.int64)
        self._call("compact", _p(ids), len(ids), _p(self._counts(starts, len(ids))), _p(flat), _p(ends))

    def trim(self, seqs) -> None:
        ids = self._ids(seqs)
        self._call("trim", _p(ids), len(ids))

    def free(self, seqs) -> None:
        ids = self._ids(seqs)
        self._call("free", _p(ids), len(ids))

    def undo(self) -> None:
        """Take back the last extend, fork or compact, if no other call that changes the table
        came after it."""
        self._call("undo")

    def moves(self) -> tuple[np.ndarray, np.ndarray]:
        """(groups [g + 1], moves [m, 2]) that the last call makes rows move by."""
        g, m = ctypes.c_int32(), ctypes.c_int32()
        self._call("moves", ctypes.addressof(g), ctypes.addressof(m))
        out = np.zeros(g.value + 1 + 2 * m.value, np.int32)
        if g.value:
            self._call("copy_moves", _p(out))
        return out[:g.value + 1], out[g.value + 1:].reshape(-1, 2)

    def table(self, seqs) -> tuple[np.ndarray, np.ndarray]:
        ids = self._ids(seqs)
        width = self._lib.rspx_pages_width(self.handle, _p(ids), len(ids))
        if width < 0:
            self.refuse("tables", width)
        table, lens = np.empty((len(ids), width), np.int32), np.empty(len(ids), np.int32)
        self._call("table", _p(ids), len(ids), width, _p(table), _p(lens))
        return table, lens

    def slots(self, seqs, first, count) -> np.ndarray:
        ids = self._ids(seqs)
        lo, n = self._counts(first, len(ids)), self._counts(count, len(ids))
        if len(n) and (n.min() < 0 or any(c > self.length(s) for s, c in zip(ids.tolist(), n.tolist()))):
            raise ValueError("PagedKVCache.slots: rows past a sequence's end")
        out = np.empty(int(n.sum()), np.int32)
        self._call("slots", _p(ids), len(ids), _p(lo), _p(n), _p(out))
        return out


class PagedKVCache:
    """``pages`` pages of ``page`` rows (a power of two), at most ``sequences`` sequences at a
    time.  Sequences are named by the numbers that ``add`` and ``fork`` give.  The methods
    keep books on the host and enqueue their copies on the current stream; those that do
    cannot be captured into a graph.  Pages given back are taken again at once: calls that
    still read them have to be on the same stream, or waited for.  A call that is refused
    (``ValueError``; ``RuntimeError`` for too few pages or sequences) or whose copies cannot be
    enqueued changes nothing.  One thread at a time."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page: int = 64, device="cuda",
                 sequences: int = 1024):
        if layers < 1 or kv_heads < 1 or head_dim < 8 or head_dim % 8:
            raise ValueError("PagedKVCache: layers and kv_heads >= 1 and head_dim a multiple of 8")
        self._t = PageTable(pages, page, sequences)
        self.layers, self.HK, self.D, self.page, self.pages = layers, kv_heads, head_dim, page, pages
        shape = (kv_heads, pages * page, head_dim)
        self.k = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(layers)]
        self.device = self.k[0].device
        bases = torch.tensor([t.data_ptr() for kv in zip(self.k, self.v) for t in kv], dtype=torch.int64).to(self.device)
        k0 = self.k[0]
        self._pool = (bases, kv_heads, head_dim, k0.stride(0), k0.stride(1), pages * page)

    @property
    def free_pages(self) -> int:
        return self._t.available

    def length(self, seq: int) -> int:
        return self._t.length(seq)

    def _done(self, what: str, y):
        """What a native call returned, unless that is a status: then raise it."""
        if y.__class__ is int:
            self._t.refuse(what, y)
        return y

    def _check_capture(self) -> None:
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("PagedKVCache: the bookkeeping cannot be captured into a graph")

    def _upload(self, *parts: np.ndarray) -> torch.Tensor:
        """int32 arrays, one after the other, on the GPU (torch keeps the pinned memory until
        the copy is done)."""
        host = torch.empty(sum(p.size for p in parts), dtype=torch.int32, pin_memory=True)
        np.concatenate([p.reshape(-1) for p in parts], out=host.numpy())
        with torch.cuda.device(self.device):
            return host.to(self.device, non_blocking=True)

    def _move_rows(self) -> None:
        """``_move``; where it fails (no memory for the lists, a refused launch) the call is taken
        back."""
        try:
            self._move()
        except BaseException:
            self._t.undo()
            raise

    def _move(self) -> None:
        """Enqueue the moves of the call just made."""
        groups, moves = self._t.moves()
        if len(groups) == 1:
            return
        flat = self._upload(groups, moves)
        bases, HK, D, sh, sn, cap = self._pool
        with torch.cuda.device(self.device):
            rc = _lib.lib().rspx_kv_move(bases.data_ptr(), bases.numel(), HK, D, sh, sn, cap, flat.data_ptr(),
                                         len(groups) - 1, flat.data_ptr() + 4 * len(groups), len(moves),
                                         _lib.stream_ptr(bases.device))
        _lib.check("rspx_kv_move", rc)

    # ------------------------------------------------------------------ sequences

    def add(self, lengths) -> list[int]:
        """New sequences of ``lengths`` rows each, whose content the caller writes."""
        return self._t.add(lengths)

    def extend(self, seqs, n=1) -> None:
        """Room for ``n`` (one number, or one per sequence) further rows of each sequence, whose
        content the caller writes.  A begun page that is shared is copied first."""
        y = _lib.calls().pages_extend(self._t.handle, seqs, n, *self._pool)
        if y is None:
            self._check_capture()
            self._t.extend(seqs, n)
            self._move_rows()
        else:
            self._done("extend", y)

    def fork(self, seqs, copies: int = 1) -> list[int]:
        """``copies`` new sequences with the content of each of ``seqs``, those of the first one
        first.  Full pages are shared; the rows of a begun page are copied."""
        y = _lib.calls().pages_fork(self._t.handle, seqs, copies, *self._pool)
        if y is None:
            self._check_capture()
            y = self._t.fork(seqs, copies)
            self._move_rows()
        return self._done("fork", y)

    def compact(self, seqs, starts, paths) -> None:
        """The accepted path of each sequence's verified trie (kv_buffer.KVCache.compact for
        many sequences): rows start + path[i] move to start + i, and the sequence ends
        after them.  ``starts``: one number or one per sequence; paths increase.  The pages
        behind the new end stay with the sequence for its next rows (``trim``)."""
        y = _lib.calls().pages_compact(self._t.handle, seqs, starts, paths, *self._pool)
        if y is None:
            self._check_capture()
            self._t.compact(seqs, starts, paths)
            self._move_rows()
        else:
            self._done("compact", y)

    def trim(self, seqs) -> None:
        """Give back the pages past each sequence's end."""
        self._t.trim(seqs)

    def free(self, seqs) -> None:
        """Forget the sequences and give back their pages."""
        y = _lib.calls().pages_free(self._t.handle, seqs)
        if y is None:
            self._t.free(seqs)
        else:
            self._done("free", y)

    # ------------------------------------------------------------------ rows

    def tables(self, seqs) -> tuple[torch.Tensor, torch.Tensor]:
        """(table [B, width] int32, lens [B] int32) on the GPU, as ``paged_attn`` takes them;
        entries past a sequence's pages are -1."""
        y = _lib.calls().pages_tables(self._t.handle, seqs, *self._pool)
        if y is not None:
            return self._done("tables", y)
        self._check_capture()
        table, lens = self._t.table(seqs)
        flat = self._upload(table, lens)
        return flat[:table.size].view(table.shape), flat[table.size:]

    def slots(self, seqs, first, count) -> torch.Tensor:
        """Pool rows (device int32) of rows first[s] .. first[s] + count[s] - 1 of each
        sequence, one sequence after the other."""
        y = _lib.calls().pages_slots(self._t.handle, seqs, first, count, *self._pool)
        if y is not None:
            return self._done("slots", y)
        self._check_capture()
        return self._upload(self._t.slots(seqs, first, count))

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """k / v [T, HK, D] bf16 of one layer to the pool rows ``slots`` [T] (device int32, as
        ``slots`` gives them; one named twice keeps parts of either row).  Can be captured."""
        T = k.shape[0]
        if tuple(k.shape) != (T, self.HK, self.D) or v.shape != k.shape or tuple(slots.shape) != (T,):
            raise ValueError(f"PagedKVCache: k and v must be [T, {self.HK}, {self.D}], slots [T]")
        fits_32_bits("PagedKVCache.write", T)
        if slots.dtype != torch.int32:
            raise TypeError("PagedKVCache: slots must be int32")
        k, v, slots = as_kernel_input(k, "k"), as_kernel_input(v, "v"), slots.contiguous()
        ck, cv = self.k[layer], self.v[layer]
        if any(t.device != ck.device for t in (k, v, slots)):
            raise RuntimeError("PagedKVCache: k, v and slots must be on the cache's GPU")
        with torch.cuda.device(self.device):
            rc = _lib.lib().rspx_kv_write(
                k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(), T,
                self.pages * self.page, ck.data_ptr(), ck.stride(0), ck.stride(1), cv.data_ptr(), cv.stride(0),
                cv.stride(1), self.HK, self.D, _lib.stream_ptr(ck.device))
        _lib.check("rspx_kv_write", rc)
