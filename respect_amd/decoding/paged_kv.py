"""KV cache of many sequences in pages: taken, shared, copied, compacted and given back.

No counterpart in the reference, whose buffer holds one request (kv_buffer.py here).
Per layer one bf16 pool [HK, pages * page, D] for K and one for V; row j of a sequence is
pool row ``table[j // page] * page + j % page``.  Who holds which page is kept on the
host (pages are counted, so that forks share the full ones); the rows move on the GPU, all
layers and sequences in one launch (rspx_kv_move).  ``paged_attn`` reads the pools through
``tables``.
"""
from __future__ import annotations

import numpy as np
import torch

from .. import _lib
from ..kernels._tensor import as_kernel_input


class PagedKVCache:
    """``pages`` pages of ``page`` rows (a power of two), at most ``sequences`` sequences at a
    time.  The bookkeeping methods run on the host, enqueue their copies on the current
    stream and cannot be captured into a graph; on a failure (``RuntimeError`` for too few
    pages or sequences, ``ValueError`` for the rest) nothing has changed."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page: int = 64, device="cuda",
                 sequences: int = 1024):
        if layers < 1 or kv_heads < 1 or pages < 1 or sequences < 1 or head_dim < 8 or head_dim % 8:
            raise ValueError("PagedKVCache: layers, kv_heads, pages, sequences >= 1 and head_dim a multiple of 8")
        if page < 1 or page & (page - 1) or pages * page >= 1 << 31:
            raise ValueError("PagedKVCache: page must be a power of two, pages * page below 2^31")
        self.layers, self.HK, self.D, self.page, self.pages = layers, kv_heads, head_dim, page, pages
        self.device = torch.device(device)
        shape = (kv_heads, pages * page, head_dim)
        self.k = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(layers)]
        self.bases = torch.tensor([t.data_ptr() for kv in zip(self.k, self.v) for t in kv], dtype=torch.int64).to(device)
        self._refs = np.zeros(pages, np.int32)                 # sequences that hold each page
        self._table = np.full((sequences, 8), -1, np.int32)    # pages of each sequence
        self._held = np.zeros(sequences, np.int64)             # how many of them
        self._len = np.full(sequences, -1, np.int64)           # rows, -1: no such sequence

    # ------------------------------------------------------------------ what is there

    @property
    def free_pages(self) -> int:
        return int((self._refs == 0).sum())

    def length(self, seq: int) -> int:
        return int(self._len[self._ids([seq])[0]])

    def _ids(self, seqs, distinct: bool = True) -> np.ndarray:
        ids = np.asarray(list(seqs), dtype=np.int64)
        if ids.size and (ids.min() < 0 or ids.max() >= len(self._len) or (self._len[ids] < 0).any()):
            raise ValueError("PagedKVCache: no such sequence")
        if distinct and len(np.unique(ids)) != len(ids):
            raise ValueError("PagedKVCache: a sequence is named twice")
        return ids

    def _counts(self, n, ids: np.ndarray) -> np.ndarray:
        c = np.broadcast_to(np.asarray(n, dtype=np.int64), ids.shape)
        if c.size and c.min() < 0:
            raise ValueError("PagedKVCache: counts must be >= 0")
        return c

    def _take(self, n: int) -> np.ndarray:
        """The n lowest free pages (not yet counted)."""
        free = np.flatnonzero(self._refs == 0)
        if len(free) < n:
            raise RuntimeError(f"PagedKVCache: {n} pages needed, {len(free)} free")
        return free[:n]

    def _new_ids(self, n: int) -> np.ndarray:
        free = np.flatnonzero(self._len < 0)
        if len(free) < n:
            raise RuntimeError(f"PagedKVCache: {n} sequences more than the {len(self._len)} there may be")
        return free[:n]

    def _widen(self, width: int) -> None:
        if width > self._table.shape[1]:
            wide = np.full((len(self._table), max(width, 2 * self._table.shape[1])), -1, np.int32)
            wide[:, :self._table.shape[1]] = self._table
            self._table = wide

    def _upload(self, *parts: np.ndarray) -> torch.Tensor:
        """int32 arrays, one after the other, on the GPU (torch keeps the pinned memory until
        the copy is done)."""
        self._check_capture()
        host = torch.empty(sum(p.size for p in parts), dtype=torch.int32, pin_memory=True)
        np.concatenate([p.reshape(-1) for p in parts], out=host.numpy(), casting="unsafe")
        with torch.cuda.device(self.device):
            return host.to(self.device, non_blocking=True)

    def _check_capture(self) -> None:
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("PagedKVCache: the bookkeeping cannot be captured into a graph")

    def tables(self, seqs) -> tuple[torch.Tensor, torch.Tensor]:
        """(table [B, width] int32, lens [B] int32) on the GPU, as ``paged_attn`` takes them;
        entries past a sequence's pages are -1."""
        ids = self._ids(seqs, distinct=False)
        width = int(self._held[ids].max(initial=0))
        flat = self._upload(self._table[ids, :width], self._len[ids])
        n = len(ids) * width
        return flat[:n].view(len(ids), width), flat[n:]

    def slots(self, seqs, first, count) -> torch.Tensor:
        """Pool rows (device int32) of rows first[s] .. first[s] + count[s] - 1 of each
        sequence, one sequence after the other."""
        ids = self._ids(seqs, distinct=False)
        lo, n = self._counts(first, ids), self._counts(count, ids)
        if (lo + n > self._len[ids]).any():
            raise ValueError("PagedKVCache: rows past a sequence's end")
        return self._upload(self._rows(ids, lo, n))

    def _rows(self, ids, lo, n) -> np.ndarray:
        s = np.repeat(ids, n)
        j = np.arange(len(s)) - np.repeat(np.cumsum(n) - n, n) + np.repeat(lo, n)
        return self._table[s, j // self.page].astype(np.int64) * self.page + j % self.page

    # ------------------------------------------------------------------ sequences

    def add(self, lengths) -> list[int]:
        """New sequences of ``lengths`` rows each, whose content the caller writes."""
        n = np.asarray(list(lengths), dtype=np.int64)
        if n.size and n.min() < 0:
            raise ValueError("PagedKVCache: counts must be >= 0")
        ids, need = self._new_ids(len(n)), -(-n // self.page)
        pages = self._take(int(need.sum()))
        self._widen(int(need.max(initial=0)))
        self._give(ids, np.zeros_like(need), need, pages)
        self._len[ids] = n
        return ids.tolist()

    def _give(self, ids, held, need, pages) -> None:
        """Sequence ids[i] gets need[i] of ``pages`` after its held[i] ones."""
        s = np.repeat(ids, need)
        at = np.arange(len(s)) - np.repeat(np.cumsum(need) - need, need) + np.repeat(held, need)
        self._table[s, at] = pages
        self._refs[pages] += 1
        self._held[ids] = held + need

    def extend(self, seqs, n=1) -> None:
        """Room for ``n`` (one number, or one per sequence) further rows of each sequence, whose
        content the caller writes.  A begun page that is shared is copied first."""
        ids = self._ids(seqs)
        n = self._counts(n, ids)
        new = self._len[ids] + n
        need = np.maximum(-(-new // self.page) - self._held[ids], 0)
        own = self._shared(ids, self._len[ids], new)
        if len(own[0]):
            self._check_capture()
        pages = self._take(int(need.sum()) + len(own[0]))
        self._widen(int((self._held[ids] + need).max(initial=0)))
        self._own(own, pages[:len(own[0])])
        self._give(ids, self._held[ids], need, pages[len(own[0]):])
        self._len[ids] = new

    def _shared(self, ids, lo, hi) -> tuple[np.ndarray, np.ndarray]:
        """(sequence, place) of the held pages with rows in [lo, hi) that others hold too."""
        first, last = lo // self.page, np.minimum(-(-hi // self.page), self._held[ids])
        n = np.where(hi > lo, np.maximum(last - first, 0), 0)
        s = np.repeat(ids, n)
        at = np.arange(len(s)) - np.repeat(np.cumsum(n) - n, n) + np.repeat(first, n)
        keep = self._refs[self._table[s, at]] > 1
        return s[keep], at[keep]

    def _own(self, own, pages) -> None:
        """Give each (sequence, place) a page of its own, with the rows of the one it shares."""
        s, at = own
        if not len(s):
            return
        old = self._table[s, at].astype(np.int64)
        rows = np.clip(self._len[s] - at * self.page, 0, self.page)
        self._move(old * self.page, pages * self.page, rows)
        np.subtract.at(self._refs, old, 1)
        self._refs[pages] += 1
        self._table[s, at] = pages

    def fork(self, seqs, copies: int = 1) -> list[int]:
        """``copies`` new sequences with the content of each of ``seqs``, those of the first one
        first.  Full pages are shared; the rows of a begun page are copied."""
        ids = self._ids(seqs, distinct=False)
        if copies < 0:
            raise ValueError("PagedKVCache: counts must be >= 0")
        src = np.repeat(ids, copies)
        new, n = self._new_ids(len(src)), self._len[src]
        full, part = n // self.page, n % self.page
        begun = np.flatnonzero(part)
        if len(begun):
            self._check_capture()
        pages = self._take(len(begun))
        width = int((full + (part > 0)).max(initial=0))
        rows = self._table[src, :width]
        rows[np.arange(width)[None] >= full[:, None]] = -1
        np.add.at(self._refs, rows[rows >= 0], 1)
        self._refs[pages] += 1
        self._move(self._table[src[begun], full[begun]].astype(np.int64) * self.page, pages * self.page, part[begun])
        rows[begun, full[begun]] = pages
        self._table[new] = -1
        self._table[new, :width] = rows
        self._held[new] = full + (part > 0)
        self._len[new] = n
        return new.tolist()

    def compact(self, seqs, starts, paths) -> None:
        """The accepted path of each sequence's verified trie (kv_buffer.KVCache.compact for
        many sequences): rows start + path[i] move to start + i, and the sequence ends
        after them.  ``starts``: one number or one per sequence; paths increase.  The pages
        behind the new end stay with the sequence for its next rows (``trim``)."""
        ids = self._ids(seqs)
        starts = self._counts(starts, ids)
        paths = [np.asarray(list(p), dtype=np.int64) for p in paths]
        if len(paths) != len(ids):
            raise ValueError("PagedKVCache: one path per sequence")
        n = np.array([len(p) for p in paths], dtype=np.int64)
        path = np.concatenate(paths) if len(paths) else np.zeros(0, np.int64)
        last = np.cumsum(n)
        seq = np.repeat(np.arange(len(ids)), n)
        inner = np.ones(len(path), bool)
        inner[(last - n)[n > 0]] = False                       # a path's first node follows none
        if (path < 0).any() or (np.diff(path, prepend=0)[inner] <= 0).any():
            raise ValueError("PagedKVCache: paths must increase")
        end = starts.copy()
        end[n > 0] += path[last[n > 0] - 1] + 1
        if (end > self._len[ids]).any():
            raise ValueError("PagedKVCache: a path runs past its sequence's end")
        to = np.arange(len(path)) - np.repeat(last - n, n)
        away = path != to                                      # the rows that do move
        lo = starts + np.bincount(seq[~away], minlength=len(ids)).astype(np.int64)
        own = self._shared(ids, lo, starts + n)
        if len(own[0]) or away.any():
            self._check_capture()
        self._own(own, self._take(len(own[0])))
        if away.any():
            s, base = ids[seq[away]], starts[seq[away]]
            a, b = base + path[away], base + to[away]
            moves = np.stack((self._table[s, a // self.page].astype(np.int64) * self.page + a % self.page,
                              self._table[s, b // self.page].astype(np.int64) * self.page + b % self.page), 1)
            count = np.bincount(seq[away], minlength=len(ids))
            self._launch(moves, count[count > 0])
        self._len[ids] = starts + n

    def trim(self, seqs) -> None:
        """Give back the pages past each sequence's end."""
        ids = self._ids(seqs)
        self._drop(ids, -(-self._len[ids] // self.page))

    def free(self, seqs) -> None:
        """Forget the sequences and give back their pages."""
        ids = self._ids(seqs)
        self._drop(ids, np.zeros(len(ids), np.int64))
        self._len[ids] = -1

    def _drop(self, ids, keep) -> None:
        width = int(self._held[ids].max(initial=0))
        rows, place = self._table[ids, :width], np.arange(width)[None]
        gone = (place >= keep[:, None]) & (place < self._held[ids][:, None])
        np.subtract.at(self._refs, rows[gone], 1)
        rows[gone] = -1
        self._table[ids, :width] = rows
        self._held[ids] = np.minimum(keep, self._held[ids])

    # ------------------------------------------------------------------ rows

    def _move(self, src, dst, rows) -> None:
        """rows[i] rows from pool row src[i] to dst[i], each run a group of its own."""
        src, dst, rows = src[rows > 0], dst[rows > 0], rows[rows > 0]
        if len(rows):
            j = np.arange(int(rows.sum())) - np.repeat(np.cumsum(rows) - rows, rows)
            self._launch(np.stack((np.repeat(src, rows) + j, np.repeat(dst, rows) + j), 1), rows)

    def _launch(self, moves: np.ndarray, count: np.ndarray) -> None:
        k0 = self.k[0]
        with torch.cuda.device(self.device):
            flat = self._upload(np.concatenate(([0], np.cumsum(count))), moves)
            rc = _lib.lib().rspx_kv_move(
                self.bases.data_ptr(), 2 * self.layers, self.HK, self.D, k0.stride(0), k0.stride(1),
                self.pages * self.page, flat.data_ptr(), len(count), flat.data_ptr() + 4 * (len(count) + 1), len(moves),
                _lib.stream_ptr(self.device))
        _lib.check("rspx_kv_move", rc)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """k / v [T, HK, D] bf16 of one layer to the pool rows ``slots`` [T] (device int32, as
        ``slots`` gives them).  Can be captured."""
        T = k.shape[0]
        if tuple(k.shape) != (T, self.HK, self.D) or v.shape != k.shape or tuple(slots.shape) != (T,):
            raise ValueError(f"PagedKVCache: k and v must be [T, {self.HK}, {self.D}], slots [T]")
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
