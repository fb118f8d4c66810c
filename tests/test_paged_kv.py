"""The paged KV cache (decoding.paged_kv): its bookkeeping on the CPU against a plain model of
it (who holds which page, lowest page first, full pages shared), and on the GPU its rows after
random runs of add, extend, write, fork, compact, trim and free against plain tensors."""
import ctypes
import random

import numpy as np
import pytest
import torch

BF = torch.bfloat16


def _table(pages, page, sequences=64):
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PageTable
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    return PageTable(pages, page, sequences)


def _pages(t, s):
    return [p for p in t.table([s])[0][0].tolist() if p >= 0]


def _moves(t):
    groups, moves = t.moves()
    assert (np.diff(groups) > 0).all() and groups[0] == 0 and groups[-1] == len(moves)
    return moves.tolist(), np.diff(groups).tolist()


def test_add_extend_fork_free():
    t = _table(12, 4)
    a, b = t.add([9, 4])
    assert (a, b) == (0, 1) and _pages(t, a) == [0, 1, 2] and _pages(t, b) == [3] and t.available == 8
    t.extend([b], 1)
    assert _pages(t, b) == [3, 4] and t.length(b) == 5
    t.extend([a, b], [3, 0])
    assert _pages(t, a) == [0, 1, 2] and t.length(a) == 12 and _moves(t) == ([], [])
    f = t.fork([b, a], 2)
    assert f == [2, 3, 4, 5]
    assert [_pages(t, s) for s in f] == [[3, 5], [3, 6], [0, 1, 2], [0, 1, 2]]
    assert _moves(t) == ([[16, 20], [16, 24]], [1, 1])
    assert t.available == 5
    t.free([a, f[0]])
    assert _moves(t) == ([], [])
    assert t.available == 6 and t.add([1]) == [0] and _pages(t, 0) == [5]
    with pytest.raises(ValueError):
        t.length(f[0])
    table, lens = t.table([b, f[2], f[1], b])
    assert table.tolist() == [[3, 4, -1], [0, 1, 2], [3, 6, -1], [3, 4, -1]] and lens.tolist() == [5, 12, 5, 5]
    assert t.slots([f[2], b], [3, 0], [2, 5]).tolist() == [3, 4, 12, 13, 14, 15, 16]
    assert t.table([])[0].shape == (0, 0) and t.slots([], 0, 0).tolist() == []


def test_compact_and_shared_pages():
    t = _table(20, 4)
    a, = t.add([13])
    t.compact([a], 6, [[0, 2, 5]])               # rows 8, 11 -> 7, 8; row 6 stays
    assert _moves(t) == ([[8, 7], [11, 8]], [2])
    assert t.length(a) == 9 and _pages(t, a) == [0, 1, 2, 3]
    t.trim([a])
    assert _pages(t, a) == [0, 1, 2]
    b, = t.fork([a], 1)                          # pages 0, 1 shared, the begun one copied
    assert _pages(t, b) == [0, 1, 3] and _moves(t)[0] == [[8, 12]]
    t.compact([b], 5, [[1]])                     # row 6 -> 5 of a page that a holds too: a new page
    assert _moves(t) == ([[6, 17], [4, 16]], [2])
    assert _pages(t, b) == [0, 4, 3] and _pages(t, a) == [0, 1, 2] and t.length(b) == 6
    d, = t.fork([a], 1)
    t.compact([d], 2, [[]])                      # cut back into a shared page
    assert t.length(d) == 2 and _moves(t) == ([], [])
    t.extend([d], 3)
    new = _pages(t, d)[0]
    assert new != 0 and _moves(t)[0] == [[0, 4 * new], [1, 4 * new + 1]] and t.length(d) == 5
    t.free([a, b, d])
    assert t.available == 20


def test_all_who_share_a_page_move_away_from_it():
    """Both holders of a page compact into it in one call: neither writes what the other reads."""
    t = _table(9, 4)
    a, = t.add([8])
    b, = t.fork([a], 1)
    t.compact([a, b], [0, 4], [[1, 2, 7], [3]])
    moves, count = _moves(t)
    assert count == [3, 1]
    old = set(range(8))
    assert {m[0] for m in moves} <= old and not {m[1] for m in moves} & old
    assert t.available == 9 - 3 - 1 and sorted(_pages(t, a) + _pages(t, b)) == [0, 1, 2, 3]
    assert t.available + len(set(_pages(t, a) + _pages(t, b))) == 9
    t.free([a, b])
    assert t.available == 9


def test_failures_change_nothing():
    t = _table(6, 4, sequences=3)
    a, b = t.add([7, 9])
    f = []

    def state():
        live = [a, b] + f
        table, lens = t.table(live)
        return table.tolist(), lens.tolist(), t.available
    before = state()
    for call in (lambda: t.add([5]), lambda: t.extend([a, b], 8), lambda: t.fork([a], 2), lambda: t.add([0, 0]),
                 lambda: t.extend([a], 1 << 40), lambda: t.add([1 << 40]), lambda: t.fork([a], 1 << 30)):
        with pytest.raises(RuntimeError):
            call()
        assert state() == before
    for call in (lambda: t.add([-1]), lambda: t.extend([a], -1), lambda: t.extend([a, a], 1), lambda: t.free([a, a]),
                 lambda: t.free([2]), lambda: t.free([-1]), lambda: t.extend([99], 1), lambda: t.fork([a], -1),
                 lambda: t.compact([a], 3, [[0, 4]]), lambda: t.compact([a], 3, [[1, 1]]),
                 lambda: t.compact([a, b], 3, [[0]]), lambda: t.compact([a], 8, [[]]), lambda: t.compact([a], 0, [[-1]]),
                 lambda: t.slots([a], 5, 3), lambda: t.slots([a], 8, 0), lambda: t.compact([a, b], [0, 1], [[2, 1], [0]]),
                 lambda: t.extend([a, b], [1]), lambda: t.free([1 << 40]), lambda: t.length(-1), lambda: t.length(1 << 40)):
        with pytest.raises(ValueError):
            call()
        assert state() == before
    assert t.fork([a, b], 0) == [] and t.add([]) == [] and state() == before
    # A full page is shared without any to spare; a begun one is not.
    c, = t.fork([b], 1)
    f.append(c)
    with pytest.raises(RuntimeError):
        t.extend([a], 2)
    from respect_amd.decoding.paged_kv import PagedKVCache
    for bad in (dict(pages=0), dict(page=3), dict(pages=1 << 28), dict(head_dim=12), dict(layers=0), dict(sequences=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(layers=1, kv_heads=1, head_dim=8, pages=4, page=16, device="cpu"), **bad})


def test_numbers_that_are_not_whole_are_refused():
    """Fractions are refused, not cut; whole numbers of any kind are taken."""
    t = _table(12, 4)
    a, b = t.add(np.array([7, 9], np.int16))
    before = t.table([a, b])[0].tolist()
    for call in (lambda: t.add([1.5]), lambda: t.extend([a], 1.9), lambda: t.extend([a, b], [1, 1.0]), lambda: t.extend([0.9], 1),
                 lambda: t.fork([0.9], 1), lambda: t.fork([a], 1.5), lambda: t.compact([a], 1.7, [[0]]),
                 lambda: t.compact([a], 1, [[0.2, 1.9]]), lambda: t.trim([0.9]), lambda: t.free([0.9]), lambda: t.table([0.9]),
                 lambda: t.slots([a], 0.5, 1), lambda: t.slots([a], 0, 1.5), lambda: t.length(0.9), lambda: t.extend(["0"], 1),
                 lambda: t.extend([a], np.array(1.5)), lambda: t.extend([a], np.array([1.5])), lambda: t.extend([a], None),
                 lambda: t.extend([a], torch.tensor([1.5]))):
        with pytest.raises((TypeError, ctypes.ArgumentError)):
            call()
        assert t.table([a, b])[0].tolist() == before and (t.length(a), t.length(b), t.available) == (7, 9, 7)
    t.extend(torch.tensor([a, b]), np.array(1))
    t.extend((a, b), torch.tensor([1, 2]))
    t.extend(iter([a]), np.int32(1))
    t.compact(np.array([a]), np.array([2]), [range(1, 3)])
    assert (t.length(a), t.length(b)) == (4, 12) and t.slots([a], torch.tensor(0), 4).tolist() == [0, 1, 2, 3]


def test_sizes_past_32_bits_are_refused():
    for sizes in ((1 << 32 | 5, 4, 8), (5, 1 << 32 | 4, 8), (5, 4, 1 << 32 | 8), (5, 4, 1 << 31), (-5, 4, 8), (5 - (1 << 32), 4, 8)):
        with pytest.raises(ValueError):
            _table(*sizes)
    with pytest.raises(TypeError):
        _table(5.5, 4, 8)


def test_random_bookkeeping_keeps_count():
    """Random calls: every page is held by as many as the count says, and never written by a move
    that another sequence's rows depend on."""
    rng = random.Random(3)
    t = _table(40, 4, sequences=12)
    live = {}                                    # sequence -> its rows' tokens
    pool, fresh = [None] * 160, iter(range(10 ** 9))

    def run_moves():
        groups, moves = t.moves()
        before = list(pool)                      # different groups: in any order
        for g in rng.sample(range(len(groups) - 1), len(groups) - 1):
            mine = moves[groups[g]:groups[g + 1]].tolist()
            for i, (src, dst) in enumerate(mine):
                assert all(dst != s for s, _ in mine[i + 1:])
                assert pool[src] == before[src] or any(dst2 == src for _, dst2 in mine[:i])
                pool[dst] = pool[src]
    for _ in range(400):
        some = rng.sample(sorted(live), rng.randint(0, len(live)))
        what = rng.choice(["add", "extend", "fork", "compact", "compact", "trim", "free"])
        try:
            if what == "add":
                n = [rng.randint(0, 11) for _ in range(2)]
                for s, k in zip(t.add(n), n):
                    live[s] = [next(fresh) for _ in range(k)]
                    for slot, x in zip(t.slots([s], 0, k), live[s]):
                        pool[slot] = x
            elif what == "extend":
                n = [rng.randint(0, 6) for _ in some]
                t.extend(some, n)
                run_moves()
                for s, k in zip(some, n):
                    new = [next(fresh) for _ in range(k)]
                    for slot, x in zip(t.slots([s], len(live[s]), k), new):
                        pool[slot] = x
                    live[s] = live[s] + new
            elif what == "fork":
                for i, s in enumerate(t.fork(some[:2], 2)):
                    live[s] = list(live[some[i // 2]])
                run_moves()
            elif what == "compact":
                starts = [rng.randint(0, len(live[s])) for s in some]
                paths = [sorted(rng.sample(range(len(live[s]) - a), rng.randint(0, len(live[s]) - a))) for s, a in zip(some, starts)]
                t.compact(some, starts, paths)
                run_moves()
                for s, a, q in zip(some, starts, paths):
                    live[s] = live[s][:a] + [live[s][a + i] for i in q]
            elif what == "trim":
                t.trim(some)
            else:
                t.free(some[:1])
                for s in some[:1]:
                    del live[s]
        except RuntimeError:
            pass                                 # full
        held = set()
        for s, rows in live.items():
            assert t.length(s) == len(rows) and [pool[x] for x in t.slots([s], 0, len(rows))] == rows
            held |= set(_pages(t, s))
        assert t.available == 40 - len(held)
    t.free(list(live))
    assert t.available == 40


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
    assert L.rspx_pages_new(0, 4, 1) is None and L.rspx_pages_new(4, 3, 1) is None and L.rspx_pages_new(4, 4, 0) is None
    assert L.rspx_pages_new(1 << 28, 16, 1) is None
    assert L.rspx_pages_add(None, None, 0, None) == -1 and L.rspx_pages_available(None) == -1
    assert L.rspx_pages_length(None, 0) == -1
    p = L.rspx_pages_new(4, 4, 2)
    assert L.rspx_pages_add(p, None, 1, None) == -1 and L.rspx_pages_fork(p, None, 1, 1, None) == -1
    assert L.rspx_pages_extend(p, None, -1, None) == -1 and L.rspx_pages_extend(p, None, 0, None) == 0
    L.rspx_pages_delete(p)
    L.rspx_pages_delete(None)


def test_c_refusals_of_moves_by_value():
    from respect_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    L = _lib.lib()

    def move(n_tensors=2, HK=2, D=64, sh=4096, sn=64, cap=64, groups=16, ng=1, moves=16, nm=1, bases=16):
        return L.rspx_kv_move_values(bases, n_tensors, HK, D, sh, sn, cap, groups, ng, moves, nm, None)
    assert move(n_tensors=-1) == -1 and move(HK=0) == -1 and move(cap=-1) == -1 and move(ng=-1) == -1
    assert move(nm=-1) == -1 and move(sn=32) == -1 and move(bases=0) == -1 and move(groups=0) == -1 and move(moves=0) == -1
    assert move(D=12) == -2 and move(HK=70000) == -2 and move(sh=4100) == -4 and move(sn=68) == -4
    assert move(ng=1, nm=480) == -2 and move(ng=960, nm=0) == -2 and move(nm=(1 << 31) - 1) == -2
    assert move(ng=0) == 0 and move(nm=0) == 0 and move(n_tensors=0) == 0
    assert L.rspx_values(16, -1, 16, None) == -1 and L.rspx_values(None, 1, 16, None) == -1
    assert L.rspx_values(16, 1, None, None) == -1 and L.rspx_values(16, 961, 16, None) == -2
    assert L.rspx_values(16, 1, 18, None) == -4 and L.rspx_values(None, 0, None, None) == 0


class _Model:
    """Every sequence's rows, as plain tensors [layers, 2, HK, n, D]."""

    def __init__(self, cache):
        self.c, self.rows = cache, {}

    def check(self):
        c = self.c
        table, _ = c.tables(list(self.rows))
        assert c.free_pages == c.pages - len(set(table[table >= 0].tolist()))
        for s, want in self.rows.items():
            n = c.length(s)
            assert n == want.shape[3]
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
    assert _lib.lib().rspx_kv_move(c._pool[0].data_ptr(), 4, 2, 128, k0.stride(0), k0.stride(1), 1024, flat.data_ptr(), 1,
                                   flat.data_ptr() + 8, 4, _lib.stream_ptr(c.device)) == 0
    c.write(0, torch.ones(3, 2, 128, dtype=BF, device="cuda"), torch.ones(3, 2, 128, dtype=BF, device="cuda"),
            torch.tensor([-1, 1024, 9], dtype=torch.int32, device="cuda"))
    for i, (a, b) in enumerate(zip(c.k + c.v, before)):
        b[:, 5] = b[:, 7]
        if i in (0, 2):
            b[:, 9] = 1
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("n_groups,n_moves", [(1, 479), (3, 478), (1, 1), (5, 30)])
def test_moves_by_value_are_the_moves(n_groups, n_moves):
    """Lists that go with the launch, up to the most that do, in a captured launch too (the lists
    changed behind it): the rows that the same lists on the device move.  Slots outside the
    cache are skipped, groups that reach past the moves are cut."""
    import numpy as np
    from respect_amd import _lib
    L, rng = _lib.lib(), np.random.default_rng(n_groups * 1000 + n_moves)
    HK, cap, D = 2, 1024, 64
    pools = [torch.randn(HK, cap, D, device="cuda").to(BF) for _ in range(4)]
    slots = rng.permutation(cap)
    moves = np.stack((slots[:n_moves], slots[n_moves:2 * n_moves]), 1).astype(np.int32)
    if n_moves > 4:
        moves[0, 0], moves[1, 1], moves[2, 0] = -1, cap, 1 << 30
    groups = np.concatenate(([0], np.sort(rng.integers(0, n_moves + 1, n_groups - 1)), [n_moves + 7])).astype(np.int32)
    flat = torch.from_numpy(np.concatenate((groups, moves.reshape(-1)))).cuda()

    def run(pools, call, g, m):
        bases = torch.tensor([t.data_ptr() for t in pools], device="cuda")
        p = pools[0]
        assert call(bases.data_ptr(), len(pools), HK, D, p.stride(0), p.stride(1), cap, g, n_groups, m, n_moves,
                    _lib.stream_ptr(p.device)) == 0
        return bases
    want = [t.clone() for t in pools]
    keep = run(want, L.rspx_kv_move, flat.data_ptr(), flat.data_ptr() + 4 * len(groups))
    got = [t.clone() for t in pools]
    run(got, L.rspx_kv_move_values, groups.ctypes.data, moves.ctypes.data)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert any(not torch.equal(a, b) for a, b in zip(got, pools)) or n_moves < 4
    got = [t.clone() for t in pools]
    bases = torch.tensor([t.data_ptr() for t in got], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert L.rspx_kv_move_values(bases.data_ptr(), 4, HK, D, got[0].stride(0), got[0].stride(1), cap, groups.ctypes.data,
                                     n_groups, moves.ctypes.data, n_moves, _lib.stream_ptr(got[0].device)) == 0
    groups[:], moves[:] = 0, 0
    for _ in range(3):
        for a, b in zip(got, pools):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del keep


@pytest.mark.gpu
def test_tables_and_slots_on_both_sides_of_what_goes_with_a_launch():
    """Tables and slots of up to 960 numbers and of more, several of them before any is looked at:
    what the books say, and nothing past the numbers is written."""
    import numpy as np
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(1, 1, 8, pages=1300, page=4)
    seqs = c.add([956, 3836, 1])
    took = [(s, c.tables(s), c._t.table(s)) for s in ([seqs[0]], seqs[1:2], seqs, [], seqs[2:])]
    for s, (table, lens), (want, n) in took:   # 240, 960, 2880, 0 and 2 numbers
        assert table.cpu().numpy().tolist() == want.tolist() and lens.tolist() == n.tolist()
    slots = [(k, c.slots([seqs[1]], 5, k), c._t.slots([seqs[1]], 5, k)) for k in (0, 1, 255, 256, 257, 959, 960, 961, 3000)]
    for k, got, want in slots:
        assert got.tolist() == want.tolist() and len(want) == k
    out = torch.full((1000,), 7, dtype=torch.int32, device="cuda")
    v = np.arange(960, dtype=np.int32)
    for n in (1, 300, 960):
        out.fill_(7)
        assert _lib.lib().rspx_values(v.ctypes.data, n, out.data_ptr(), _lib.stream_ptr(out.device)) == 0
        assert out[:n].tolist() == list(range(n)) and (out[n:] == 7).all()


@pytest.mark.gpu
def test_fork_on_both_sides_of_what_goes_with_a_launch():
    """Begun pages of 63 rows copied 7 and 8 times: 441 moves go with the launch, 504 do not."""
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(2, 2, 64, pages=40, page=64)
    for t in c.k + c.v:
        t.copy_(torch.randn(t.shape, device="cuda"))
    s, = c.add([127])
    want = [t[:, :127].clone() for t in c.k + c.v]
    for copies in (7, 8):
        forks = c.fork([s], copies)
        for f in forks:
            at = c.slots([f], 0, 127).long()
            assert all(torch.equal(t[:, at], w) for t, w in zip(c.k + c.v, want))
        c.free(forks)


def _books(c, seqs):
    table, lens = c._t.table(seqs)
    return table.tolist(), lens.tolist(), c.free_pages


def test_undo_after_random_calls():
    """extend, fork and compact taken back: every sequence's pages and length, the free pages and the
    numbers and pages taken next are those of a table that never saw the call."""
    def play(seed, undone):
        rng, t = random.Random(seed), _table(30, 4, sequences=10)
        live, log = [], []
        for _ in range(120):
            some = rng.sample(live, rng.randint(0, len(live)))
            what = rng.choice(["add", "extend", "extend", "fork", "compact", "compact", "trim", "free"])
            n = [rng.randint(0, 6) for _ in some]
            room = [t.length(s) for s in some]
            starts = [rng.randint(0, k) for k in room]
            paths = [sorted(rng.sample(range(k - a), rng.randint(0, k - a))) for k, a in zip(room, starts)]
            back = rng.random() < 0.4 and what in ("extend", "fork", "compact")
            if back and not undone:
                continue
            try:
                if what == "add":
                    live += t.add([rng.randint(0, 9)])
                elif what == "extend":
                    t.extend(some, n)
                elif what == "fork":
                    new = t.fork(some[:2], 2)
                    live += [] if back else new
                elif what == "compact":
                    t.compact(some, starts, paths)
                elif what == "trim":
                    t.trim(some)
                else:
                    t.free(some[:1])
                    live = [s for s in live if s not in some[:1]]
            except RuntimeError:
                continue
            if back:
                t.undo()
                assert _moves(t) == ([], [])
                t.undo()                         # and nothing more
            table, lens = t.table(live)
            log.append((back, live[:], table.tolist(), lens.tolist(), t.available))
        return [x[1:] for x in log if not x[0]], sum(x[0] for x in log)
    took = 0
    for seed in range(30):
        with_, n = play(seed, True)
        assert with_ == play(seed, False)[0]
        took += n
    assert took > 200
    t = _table(8, 4)
    t.extend(t.add([3]), 4)
    t.add([1])
    t.undo()                                     # behind an add: nothing
    assert t.length(0) == 7 and t.available == 5


def test_a_copy_that_fails_takes_the_books_back(monkeypatch):
    """The rows of a call cannot be moved (no memory for the lists, a refused launch): lengths, pages
    and free pages are as before it, and the next sequences get the numbers they would have."""
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    c = PagedKVCache(1, 1, 8, pages=20, page=4, device="cpu")
    monkeypatch.setattr(c, "_check_capture", lambda: None)
    monkeypatch.setattr(c, "_move", lambda: None)
    a, b = c.add([9, 6])
    f, = c.fork([a])
    c.compact([f], 2, [[]])                     # its next rows lie in a page that a holds too
    seqs = [a, b, f]
    before = _books(c, seqs)

    def fail():
        raise RuntimeError("out of memory")
    monkeypatch.setattr(c, "_move", fail)
    for call in (lambda: c.fork([a, b], 2), lambda: c.extend([f, a], [3, 9]), lambda: c.compact([b, f], [0, 0], [[1, 2], [1]])):
        with pytest.raises(RuntimeError, match="memory"):
            call()
        assert _books(c, seqs) == before
    monkeypatch.setattr(c, "_move", lambda: None)
    assert c.fork([b]) == [3] and c.add([0]) == [4]
    c.free([a, b, f, 3, 4])
    assert c.free_pages == 20


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("copies", [2, 60])
def test_moves_that_the_library_refuses_take_the_books_back(native, copies, monkeypatch):
    """The same with the real copies refused (a head_dim that is none), for lists that go with the
    launch and longer ones; afterwards the calls do what they should."""
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache

    class Leave:
        def __getattr__(self, name):
            return lambda *a: None
    if not native:
        monkeypatch.setattr(_lib, "_calls", Leave())
    c = PagedKVCache(2, 2, 64, pages=200, page=16)
    for t in c.k + c.v:
        t.copy_(torch.randn(t.shape, device="cuda"))
    s, u = c.add([45, 30])
    want = [t[:, :45].clone() for t in c.k + c.v]
    before, pool = _books(c, [s, u]), c._pool
    c._pool = pool[:2] + (12,) + pool[3:]
    for call in (lambda: c.fork([s], copies), lambda: c.compact([s, u], 0, [[1, 2], [3]])):
        with pytest.raises(RuntimeError):
            call()
        assert _books(c, [s, u]) == before
    c._pool = pool
    forks = c.fork([s], copies)
    assert forks == list(range(2, 2 + copies))
    for f in forks:
        at = c.slots([f], 0, 45).long()
        assert all(torch.equal(t[:, at], w) for t, w in zip(c.k + c.v, want))
    c.compact([s], 0, [[1, 2]])
    at = c.slots([s], 0, 2).long()
    assert all(torch.equal(t[:, at], w[:, 1:3]) for t, w in zip(c.k + c.v, want))
    c.free([s, u] + forks)
    assert c.free_pages == 200


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
def test_write_of_more_threads_than_a_grid_holds():
    """4097 tokens of 2^20 16-byte pieces each, 2^32 and more threads: the last token is written too.
    All are the same row, all but two go nowhere."""
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(1, 4096, 2048, pages=2, page=1)
    k, v = (torch.randn(1, 4096, 2048, device="cuda").to(BF) for _ in range(2))
    slots = torch.full((4097,), -1, dtype=torch.int32, device="cuda")
    slots[0], slots[4096] = 0, 1
    c.write(0, k.expand(4097, -1, -1), v.expand(4097, -1, -1), slots)
    for pool, x in ((c.k[0], k), (c.v[0], v)):
        assert torch.equal(pool[:, 0], x[0]) and torch.equal(pool[:, 1], x[0])


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
    c.write(0, k[:0], k[:0], slots[:0])
    table, lens = c.tables([])
    assert table.shape == (0, 0) and lens.shape == (0,) and c.slots([], 0, 0).shape == (0,)
    assert c.device.index is not None
