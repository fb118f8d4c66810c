"""The paged KV cache (decoding.paged_kv): its bookkeeping on the CPU against a plain model of
it (who holds which page, lowest page first, full pages shared), and on the GPU its rows after
random runs of add, extend, write, fork, compact, trim and free against plain tensors."""
import random

import numpy as np
import pytest
import torch

BF = torch.bfloat16


class _Dry:
    """A PagedKVCache without device work: the moves are recorded instead of launched."""

    def __new__(cls, pages, page, sequences=64):
        from respect_amd.decoding.paged_kv import PagedKVCache

        class Dry(PagedKVCache):
            def _launch(self, moves, count):
                self.moves.append((moves.copy(), count.copy()))

            def _upload(self, *parts):
                return torch.from_numpy(np.concatenate([p.reshape(-1) for p in parts]).astype(np.int32))

            def _check_capture(self):
                pass
        c = Dry(1, 1, 8, pages, page=page, device="cpu", sequences=sequences)
        c.moves = []
        return c


def _pages(c, s):
    return c._table[s, :c._held[s]].tolist()


def test_add_extend_fork_free():
    c = _Dry(12, 4)
    a, b = c.add([9, 4])
    assert (a, b) == (0, 1) and _pages(c, a) == [0, 1, 2] and _pages(c, b) == [3] and c.free_pages == 8
    c.extend([b], 1)
    assert _pages(c, b) == [3, 4] and c.length(b) == 5
    c.extend([a, b], [3, 0])
    assert _pages(c, a) == [0, 1, 2] and c.length(a) == 12 and not c.moves
    f = c.fork([b, a], 2)
    assert f == [2, 3, 4, 5]
    assert [_pages(c, s) for s in f] == [[3, 5], [3, 6], [0, 1, 2], [0, 1, 2]]
    moves, count = c.moves.pop()
    assert moves.tolist() == [[16, 20], [16, 24]] and count.tolist() == [1, 1] and not c.moves
    assert c.free_pages == 5
    c.free([a, f[0]])
    assert c.free_pages == 6 and c.add([1]) == [0] and _pages(c, 0) == [5]
    with pytest.raises(ValueError):
        c.length(f[0])
    table, lens = c.tables([b, f[2], f[1]])
    assert table.tolist() == [[3, 4, -1], [0, 1, 2], [3, 6, -1]] and lens.tolist() == [5, 12, 5]
    assert c.slots([f[2], b], [3, 0], [2, 5]).tolist() == [3, 4, 12, 13, 14, 15, 16]


def test_compact_and_shared_pages():
    c = _Dry(20, 4)
    a, = c.add([13])
    c.compact([a], 6, [[0, 2, 5]])               # rows 8, 11 -> 7, 8; row 6 stays
    moves, count = c.moves.pop()
    assert moves.tolist() == [[8, 7], [11, 8]] and count.tolist() == [2]
    assert c.length(a) == 9 and _pages(c, a) == [0, 1, 2, 3]
    c.trim([a])
    assert _pages(c, a) == [0, 1, 2]
    b, = c.fork([a])                             # pages 0, 1 shared, the begun one copied
    assert _pages(c, b) == [0, 1, 3]
    assert c.moves.pop()[0].tolist() == [[8, 12]]
    c.compact([b], 5, [[1]])                     # row 6 -> 5 of a page that a holds too
    own, path = c.moves
    assert own[0].tolist() == [[4, 16], [5, 17], [6, 18], [7, 19]] and path[0].tolist() == [[18, 17]]
    assert _pages(c, b) == [0, 4, 3] and _pages(c, a) == [0, 1, 2] and c.length(b) == 6
    c.moves.clear()
    d, = c.fork([a])
    c.compact([d], 2, [[]])                      # cut back into a shared page
    assert c.length(d) == 2
    c.moves.clear()
    c.extend([d], 3)
    new = _pages(c, d)[0]
    assert new != 0 and c.moves.pop()[0].tolist() == [[0, 4 * new], [1, 4 * new + 1]]
    assert c._refs[0] == 2 and c.length(d) == 5
    c.free([a, b, d])
    assert c.free_pages == 20


def test_failures_change_nothing():
    c = _Dry(6, 4, sequences=3)
    a, b = c.add([7, 9])
    before = (c._refs.copy(), c._table.copy(), c._held.copy(), c._len.copy())

    def same():
        return all((x == y).all() for x, y in zip(before, (c._refs, c._table, c._held, c._len)))
    for call in (lambda: c.add([5]), lambda: c.extend([a, b], 8), lambda: c.fork([a], 2), lambda: c.add([0, 0])):
        with pytest.raises(RuntimeError):
            call()
        assert same()
    for call in (lambda: c.add([-1]), lambda: c.extend([a], -1), lambda: c.extend([a, a]), lambda: c.free([a, a]),
                 lambda: c.free([2]), lambda: c.free([-1]), lambda: c.extend([99]), lambda: c.fork([a], -1),
                 lambda: c.compact([a], 3, [[0, 4]]), lambda: c.compact([a], 3, [[1, 1]]),
                 lambda: c.compact([a, b], 3, [[0]]), lambda: c.compact([a], 8, [[]]), lambda: c.compact([a], 0, [[-1]]),
                 lambda: c.slots([a], 5, 3), lambda: c.compact([a, b], [0, 1], [[2, 1], [0]])):
        with pytest.raises(ValueError):
            call()
        assert same()
    for bad in (dict(pages=0), dict(page=3), dict(pages=1 << 28), dict(head_dim=12), dict(layers=0)):
        with pytest.raises(ValueError):
            from respect_amd.decoding.paged_kv import PagedKVCache
            PagedKVCache(**{**dict(layers=1, kv_heads=1, head_dim=8, pages=4, page=16, device="cpu"), **bad})
    assert c.fork([a, b], 0) == [] and c.add([]) == [] and same()


def test_c_refusals():
    from respect_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    L = _lib.lib()

    def move(n_tensors=2, HK=2, D=64, sh=4096, sn=64, cap=64, groups=16, ng=1, moves=16, nm=1, bases=16):
        return L.rspx_kv_move(bases, n_tensors, HK, D, sh, sn, cap, groups, ng, moves, nm, None)
    assert move(n_tensors=-1) == -1 and move(HK=0) == -1 and move(cap=-1) == -1 and move(ng=-1) == -1
    assert move(nm=-1) == -1 and move(sn=32) == -1 and move(bases=0) == -1 and move(groups=0) == -1 and move(moves=0) == -1
    assert move(D=12) == -2 and move(HK=70000) == -2
    assert move(sh=4100) == -4 and move(sn=68) == -4
    assert move(ng=0) == 0 and move(nm=0) == 0 and move(n_tensors=0) == 0

    def write(p=16, T=2, cap=64, D=64, s=64, slots=16):
        return L.rspx_kv_write(p, 128, s, p, 128, 64, slots, T, cap, p, 4096, 64, p, 4096, 64, 2, D, None)
    assert write(T=-1) == -1 and write(cap=-1) == -1 and write(p=0) == -1 and write(slots=0) == -1
    assert write(D=60) == -2 and write(p=8) == -4 and write(s=68) == -4
    assert write(T=0) == 0


class _Model:
    """Every sequence's rows, as plain tensors [layers, 2, HK, n, D]."""

    def __init__(self, cache):
        self.c, self.rows = cache, {}

    def check(self):
        c = self.c
        pages = [p for s in self.rows for p in _pages(c, s)]
        assert (np.bincount(np.array(pages, dtype=int), minlength=c.pages) == c._refs).all()
        for s, want in self.rows.items():
            n = c.length(s)
            assert n == want.shape[3] and c._held[s] >= -(-n // c.page)
            slots = c.slots([s], 0, n).long()
            got = torch.stack([torch.stack((k[:, slots], v[:, slots])) for k, v in zip(c.k, c.v)])
            assert torch.equal(got.cpu(), want), f"sequence {s}"


@pytest.mark.gpu
@pytest.mark.parametrize("page,D,HK,layers", [(16, 128, 2, 3), (4, 64, 1, 2), (64, 32, 3, 1), (1, 8, 2, 2), (16, 96, 1, 1),
                                              (128, 256, 1, 2)])
def test_random_runs_against_plain_tensors(page, D, HK, layers):
    from respect_amd.decoding.paged_kv import PagedKVCache
    rng = random.Random(page + D)
    g = torch.Generator()
    g.manual_seed(page)
    c = PagedKVCache(layers, HK, D, pages=max(24, 3000 // page), page=page, sequences=24)
    m = _Model(c)

    def fill(seqs, first, count):
        new = [torch.randn(layers, 2, HK, n, D, generator=g).to(BF) for n in count]
        slots = c.slots(seqs, first, count)
        every = torch.cat(new + [torch.empty(layers, 2, HK, 0, D, dtype=BF)], 3).cuda()
        for i in range(layers):
            k, v = (t.transpose(0, 1) for t in every[i])       # head-major rows: strided
            c.write(i, k, v, slots)
        return new
    for step in range(40):
        live = sorted(m.rows)
        some = rng.sample(live, rng.randint(0, len(live)))
        what = rng.choice(["add", "extend", "fork", "compact", "compact", "trim", "free"])
        print(step, what, len(some), flush=True)
        try:
            if what == "add":
                n = [rng.randint(0, 70) for _ in range(rng.randint(1, 3))]
                seqs = c.add(n)
                for s, x in zip(seqs, fill(seqs, 0, n)):
                    m.rows[s] = x
            elif what == "extend":
                n = [rng.randint(0, 40) for _ in some]
                first = [c.length(s) for s in some]
                c.extend(some, n)
                for s, x in zip(some, fill(some, first, n)):
                    m.rows[s] = torch.cat((m.rows[s], x), 3)
            elif what == "fork" and some:
                some = some[:2]
                for i, s in enumerate(c.fork(some, 2)):
                    m.rows[s] = m.rows[some[i // 2]].clone()
            elif what == "compact":
                starts, paths = [], []
                for s in some:
                    n = c.length(s)
                    starts.append(rng.randint(0, n))
                    room = n - starts[-1]
                    paths.append(sorted(rng.sample(range(room), rng.randint(0, min(room, 30)))))
                c.compact(some, starts, paths)
                for s, a, p in zip(some, starts, paths):
                    m.rows[s] = torch.cat((m.rows[s][:, :, :, :a], m.rows[s][:, :, :, [a + i for i in p]]), 3)
            elif what == "trim":
                c.trim(some)
            elif what == "free":
                c.free(some[:3])
                for s in some[:3]:
                    del m.rows[s]
        except RuntimeError as e:
            assert "PagedKVCache" in str(e)                    # full: nothing changed
        m.check()
    c.free(list(m.rows))
    assert c.free_pages == c.pages


@pytest.mark.gpu
def test_long_groups_in_order_and_skipped_slots():
    """A path of more rows than a workgroup holds at once, moved down by one; rows outside the cache
    are neither read nor written."""
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(2, 2, 128, pages=64, page=16)
    for t in c.k + c.v:
        t.copy_(torch.randn(t.shape, device="cuda"))
    before = [t.clone() for t in c.k + c.v]
    s, = c.add([1000])
    c.compact([s], 0, [list(range(1, 1000))])
    for a, b in zip(c.k + c.v, before):
        assert torch.equal(a[:, :999], b[:, 1:1000]) and torch.equal(a[:, 999:], b[:, 999:])
    before = [t.clone() for t in c.k + c.v]
    flat = torch.tensor([0, 4, -5, 3, 3, 1 << 20, 1024, 0, 7, 5], dtype=torch.int32, device="cuda")
    k0 = c.k[0]
    assert _lib.lib().rspx_kv_move(c.bases.data_ptr(), 4, 2, 128, k0.stride(0), k0.stride(1), 1024, flat.data_ptr(), 1,
                                   flat.data_ptr() + 8, 4, _lib.stream_ptr(c.device)) == 0
    c.write(0, torch.ones(3, 2, 128, dtype=BF, device="cuda"), torch.ones(3, 2, 128, dtype=BF, device="cuda"),
            torch.tensor([-1, 1024, 9], dtype=torch.int32, device="cuda"))
    for i, (a, b) in enumerate(zip(c.k + c.v, before)):
        b[:, 5] = b[:, 7]
        if i in (0, 2):
            b[:, 9] = 1
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_capture_is_refused_and_write_is_captured():
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(1, 1, 64, pages=8, page=4)
    s, = c.add([6])
    slots = c.slots([s], 0, 6)
    k, v = (torch.randn(6, 1, 64, device="cuda").to(BF) for _ in range(2))
    c.write(0, k, v, slots)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.write(0, k, v, slots)
        for call in (lambda: c.fork([s]), lambda: c.tables([s]), lambda: c.compact([s], 0, [[1]])):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    assert c.length(s) == 6 and c.free_pages == 6
    for _ in range(3):
        k.normal_()
        g.replay()
        assert torch.equal(c.k[0][:, slots.long()], k.transpose(0, 1)) and torch.equal(c.v[0][:, slots.long()], v.transpose(0, 1))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_gpu_refusals():
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(1, 2, 64, pages=8, page=4)
    s, = c.add([6])
    slots = c.slots([s], 0, 6)
    k = torch.zeros(6, 2, 64, dtype=BF, device="cuda")
    with pytest.raises(ValueError):
        c.write(0, k[:5], k, slots)
    with pytest.raises(ValueError):
        c.write(0, k[:, :1], k[:, :1], slots)
    with pytest.raises(TypeError):
        c.write(0, k, k, slots.long())
    with pytest.raises(TypeError):
        c.write(0, k.float(), k.float(), slots)
    with pytest.raises(RuntimeError):
        c.write(0, k, k, slots.cpu())
