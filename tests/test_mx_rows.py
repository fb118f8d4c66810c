"""Rows of a cache in the microscaled formats (kernels.mx, PagedKVCache(dtype=...)) against their
definition in 64 bits: every bf16 value, groups of any scale, of zeros, infinities and NaN, bad
slots, strides, a captured call, offsets past 32 bits, moves of rows; refusals on the CPU."""
import random

import pytest
import torch

from _mx import BITS, POSITIVE, quantise, values

BF = torch.bfloat16
FORMATS = ["mxfp8", "mxfp4"]


def _lib():
    from respect_amd import _lib as L
    if not L.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    return L


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _same(a, b):
    """Equal values, NaN to NaN."""
    a, b = a.double().cpu(), b.double().cpu()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("fmt", FORMATS)
def test_the_definition(fmt):
    """Known values of the formats, on the CPU."""
    most = POSITIVE[fmt][-1]
    assert most == {"mxfp8": 448.0, "mxfp4": 6.0}[fmt]
    x = torch.zeros(7, 32)
    x[1, 3] = most
    x[2, 3] = most * 1.01
    x[3, :2] = torch.tensor([-2.0 ** -100, 2.0 ** -130])
    x[4, 5] = float("inf")
    x[5, 5] = float("nan")
    x[6] = torch.arange(32) - 16.0
    codes, scales = quantise(x.to(BF), fmt)
    assert scales[:, 0].tolist()[:6] == [10, 127, 128, {"mxfp8": 19, "mxfp4": 25}[fmt], 255, 255]
    y = values(codes, scales, fmt)
    assert (y[0] == 0).all() and y[1, 3] == most and y[4:6].isnan().all() and y[3, 0] == -2.0 ** -100
    step = {"mxfp8": 2.0 ** -4, "mxfp4": 2.0 ** -2}[fmt]              # half a step of the mantissa
    assert ((y[6] - x[6]).abs() <= step * x[6].abs() + {"mxfp8": 0.0, "mxfp4": 1.0}[fmt]).all()


def test_refusals():
    L = _lib()
    from respect_amd.decoding.paged_kv import PagedKVCache
    from respect_amd.kernels.mx import MXRows, read_rows, write_rows
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    for bad in (("mxfp6", u8(2, 8, 64), u8(2, 8, 2)), ("mxfp8", u8(2, 8, 48), u8(2, 8, 2)), ("mxfp8", u8(2, 8, 64), u8(2, 8, 1)),
                ("mxfp4", u8(2, 8, 64), u8(2, 8, 2)), ("mxfp8", u8(2, 8, 64), u8(2, 9, 2)), ("mxfp8", u8(8, 64), u8(8, 2)),
                ("mxfp8", u8(2, 8, 72)[..., :64], u8(2, 8, 2)), ("mxfp8", u8(2, 8, 80)[..., 8:72], u8(2, 8, 2)),
                ("mxfp8", u8(2, 64, 8).transpose(1, 2), u8(2, 8, 2))):
        with pytest.raises(ValueError):
            MXRows(bad[1], bad[2], bad[0])
    with pytest.raises(TypeError):
        MXRows(u8(2, 8, 64).int(), u8(2, 8, 2), "mxfp8")
    with pytest.raises(ValueError):
        MXRows.empty(2, 8, 48, "mxfp8", device="cpu")
    p, x, s = MXRows.empty(2, 8, 64, "mxfp8", device="cpu"), torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        write_rows(x, x, p, p, s)
    with pytest.raises(RuntimeError):
        read_rows(p, p, s)
    with pytest.raises(TypeError):
        write_rows(x, x, p, p, s.long())
    with pytest.raises(TypeError):
        write_rows(x, x, torch.zeros(2, 8, 64, dtype=BF), p, s)
    for args in ((x[:2], x, p, p, s), (x, x[:2], p, p, s), (x[:, :1], x[:, :1], p, p, s), (x, x, p, p, s[None]),
                 (x, x, p, MXRows.empty(2, 8, 64, "mxfp4", device="cpu"), s)):
        with pytest.raises(ValueError):
            write_rows(*args)
    for bad in (dict(dtype="fp8"), dict(dtype="mxfp8", head_dim=48), dict(dtype=None)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(layers=1, kv_heads=1, head_dim=64, pages=4, page=4, device="cpu"), **bad})
    c = PagedKVCache(2, 2, 64, pages=4, page=4, device="cpu", dtype="mxfp4")
    assert c.k[1].shape == (2, 16, 64) and c.k[0].codes.shape == (2, 16, 32) and c.v[0].scales.shape == (2, 16, 2)
    lib = L.lib()

    def write(T=2, cap=8, HK=2, D=64, fmt=8, x=16, st=128, codes=16, sn=64, scales=1, ssn=2, slots=4):
        return lib.rspx_kv_write_mx(x, st, 64, x, st, 64, slots, T, cap, codes, 512, sn, scales, 16, ssn, codes, 512, sn, scales, 16,
                                    ssn, HK, D, fmt, None)

    def read(T=2, cap=8, HK=2, D=64, fmt=8, x=16, st=128, codes=16, sn=64, scales=1, ssn=2, slots=4):
        return lib.rspx_kv_read(codes, 512, sn, scales, 16, ssn, codes, 512, sn, scales, 16, ssn, slots, T, cap, x, st, 64, x, st, 64,
                                HK, D, fmt, None)
    for f in (write, read):
        assert f(T=-1) == -1 and f(cap=-1) == -1 and f(HK=0) == -1 and f(D=0) == -1 and f(x=0) == -1 and f(slots=0) == -1
        assert f(codes=0) == -1 and f(scales=0) == -1 and f(sn=32) == -1 and f(ssn=1) == -1
        assert f(fmt=6) == -2 and f(D=72) == -2 and f(D=2080) == -2 and f(HK=70000) == -2
        assert f(x=8) == -4 and f(st=130) == -4 and f(codes=8) == -4 and f(sn=72) == -4
        assert f(T=0) == 0
    assert write(fmt=16) == -2 and read(fmt=16, sn=64, scales=0, T=0) == 0

    def move(fn, bases=16, n=2, HK=2, D=64, fmt=8, sch=512, scn=64, ssh=16, ssn=2, cap=8, groups=16, ng=1, moves=16, nm=1):
        return fn(bases, n, HK, D, fmt, sch, scn, ssh, ssn, cap, groups, ng, moves, nm, None)
    for fn in (lib.rspx_kv_move_mx, lib.rspx_kv_move_mx_values):
        assert move(fn, n=-1) == -1 and move(fn, HK=0) == -1 and move(fn, cap=-1) == -1 and move(fn, ng=-1) == -1
        assert move(fn, scn=32) == -1 and move(fn, ssn=1) == -1 and move(fn, bases=0) == -1 and move(fn, groups=0) == -1
        assert move(fn, fmt=16) == -2 and move(fn, D=72) == -2 and move(fn, HK=70000) == -2 and move(fn, n=40000) == -2
        assert move(fn, sch=520) == -4 and move(fn, scn=72) == -4
        assert move(fn, ng=0) == 0 and move(fn, nm=0) == 0 and move(fn, n=0) == 0
    assert move(lib.rspx_kv_move_mx_values, nm=480) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_value(fmt):
    """All 65536 bf16 patterns beside a largest one of each kind of mantissa and many exponents,
    infinities and NaN in groups of their own."""
    from respect_amd.kernels.mx import MXRows, read_rows, write_rows
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    finite = every[torch.isfinite(every.float())]
    for top in (1.0, 1.5, 1.5078125, 1.75, 1.7578125, 1.9921875):
        for e in (-126, -117, -100, -3, 0, 7, 60, 119, 127):
            big = torch.tensor(top * 2.0 ** e).to(BF)
            x = finite[finite.float().abs() <= big.float()]
            x = x[:len(x) // 31 * 31].view(-1, 31)
            x = torch.cat((big.expand(len(x), 1), x), 1)
            n = -(-len(x) // 4)
            rows = torch.zeros(n * 4, 32, dtype=BF)
            rows[:len(x)] = x
            rows = rows.view(n, 1, 128)
            p = MXRows.empty(1, n, 128, fmt)
            slots = torch.arange(n, dtype=torch.int32, device="cuda")
            write_rows(rows.cuda(), rows.flip(-1).cuda(), p, MXRows.empty(1, n, 128, fmt), slots)
            codes, scales = quantise(rows, fmt)
            assert torch.equal(p.scales[0].cpu(), scales[:, 0]) and torch.equal(p.codes[0].cpu(), codes[:, 0]), (top, e)
            k, _ = read_rows(p, p, slots)
            # Exact, but for what rounds up to 2^128, the first number that bf16 does not hold.
            want = values(codes, scales, fmt)
            want = torch.where(want.abs() == 2.0 ** 128, want.sign() * float("inf"), want)
            assert torch.equal(k.cpu().double(), want), (top, e)
    odd = every[~torch.isfinite(every.float())]
    x = torch.ones(len(odd), 4, 32, dtype=BF)
    x[torch.arange(len(odd)), 1, torch.arange(len(odd)) % 32] = odd
    p = MXRows.empty(1, len(odd), 128, fmt)
    slots = torch.arange(len(odd), dtype=torch.int32, device="cuda")
    write_rows(x.view(-1, 1, 128).cuda(), x.view(-1, 1, 128).cuda(), p, p, slots)
    k, v = read_rows(p, p, slots)
    assert (p.scales[0, :, 1] == 255).all() and (p.scales[0, :, [0, 2, 3]] != 255).all()
    assert k.view(-1, 4, 32)[:, 1].isnan().all() and (k.view(-1, 4, 32)[:, [0, 2, 3]] == 1).all() and _same(k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,HK,D,page", [(1, 1, 32, 1), (5, 3, 64, 4), (300, 2, 128, 16), (33, 1, 96, 16), (70, 8, 256, 64),
                                         (9, 1, 2048, 4), (4000, 8, 128, 64)])
def test_write_and_read(fmt, T, HK, D, page):
    """Rows to scattered slots, some outside the pool; what is not named stays; strided rows and
    pools; read back in another order, slots outside giving NaN."""
    from respect_amd.decoding.paged_kv import PagedKVCache
    from respect_amd.kernels.mx import MXRows, read_rows, write_rows
    g = torch.Generator().manual_seed(T + D)
    pages = -(-T // page) + 2
    c = PagedKVCache(2, HK, D, pages=pages, page=page, dtype=fmt)
    scale = torch.exp(3 * torch.randn(T, HK, D // 32, 1, generator=g))
    k, v = ((torch.randn(T, HK, D // 32, 32, generator=g) * scale).flatten(-2).to(BF) for _ in range(2))
    k[0] = 0
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    named = slots.clone()
    if T > 4:
        slots[1], slots[3] = -1, pages * page
    for t in (c.k[1], c.v[1]):
        t.codes.fill_(0x11)
        t.scales.fill_(100)
    wide = torch.zeros(2, HK, T, D + 8, dtype=BF, device="cuda")
    wide[0, :, :, :D], wide[1, :, :, :D] = k.transpose(0, 1).cuda(), v.transpose(0, 1).cuda()
    ks, vs = (w[:, :, :D].transpose(0, 1) for w in wide)
    for layer, a, b in ((1, k.cuda(), v.cuda()), (0, ks, vs)):
        c.write(layer, a, b, slots.cuda())
        for pool, x in ((c.k[layer], k), (c.v[layer], v)):
            codes, scales = quantise(x, fmt)
            want_c, want_s = torch.full_like(pool.codes, 0x11 * layer).cpu(), torch.full_like(pool.scales, 100 * layer).cpu()
            for t in range(T):
                if 0 <= slots[t] < pages * page:
                    want_c[:, slots[t]], want_s[:, slots[t]] = codes[t], scales[t]
            assert torch.equal(pool.codes.cpu(), want_c) and torch.equal(pool.scales.cpu(), want_s)
    order = torch.randperm(T, generator=g)
    at = named[order].clone()
    ok = (slots[order] == at)
    at[~ok] = -5
    got = c.read(1, at.cuda())
    for y, x in zip(got, (k, v)):
        assert y.shape == (T, HK, D) and y.dtype == BF and y.is_contiguous()
        want = values(*quantise(x, fmt), fmt)[order]
        want[~ok] = float("nan")
        assert _same(y, want)
    # Pools inside wider ones, slot-major: [slots, HK, ...].
    n, rb, sb = pages * page, D * BITS[fmt] // 8, D // 32
    base = torch.zeros(2, n, HK, rb + 16, dtype=torch.uint8, device="cuda"), torch.zeros(2, n, HK, sb + 3, dtype=torch.uint8, device="cuda")
    pk, pv = (MXRows(base[0][i].transpose(0, 1)[..., :rb], base[1][i].transpose(0, 1)[..., 1:1 + sb], fmt) for i in (0, 1))
    write_rows(k.cuda(), v.cuda(), pk, pv, slots.cuda())
    assert (base[0][..., rb:] == 0).all() and (base[1][..., 0] == 0).all() and (base[1][..., 1 + sb:] == 0).all()
    assert all(_same(a, b) for a, b in zip(read_rows(pk, pv, at.cuda()), got))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 64, 96, 128])
def test_read_of_a_bf16_cache(D):
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(1, 3, D, pages=9, page=8)
    c.k[0].copy_(torch.randn(3, 72, D, device="cuda"))
    c.v[0].copy_(torch.randn(3, 72, D, device="cuda"))
    slots = _i32([70, 0, 5, 5, 33, 72, -1])
    k, v = c.read(0, slots)
    for y, x in ((k, c.k[0]), (v, c.v[0])):
        assert torch.equal(y[:5], x[:, slots[:5].long()].transpose(0, 1)) and y[5:].isnan().all()
    assert c.read(0, slots[:0])[0].shape == (0, 3, D)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(fmt):
    """Pools whose heads and rows lie more than 2^32 bytes apart."""
    from respect_amd.kernels.mx import MXRows, read_rows, write_rows
    rb = 64 * BITS[fmt] // 8
    base = torch.zeros(2, 300, 1 << 23, dtype=torch.uint8, device="cuda")          # 5 GB
    p = MXRows(base[:, :, :rb], base[:, :, 4096:4098], fmt)
    v = MXRows(base[:, :, 8192:8192 + rb], base[:, :, 4098:4100], fmt)
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(0)).to(BF)
    slots = _i32([299, 0, 255, 298])
    write_rows(x.cuda(), x.flip(0).contiguous().cuda(), p, v, slots)
    a, b = read_rows(p, v, slots)
    want = values(*quantise(x, fmt), fmt)
    assert _same(a, want) and _same(b, want.flip(0))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_captured(fmt):
    """Two graphs of a write and a read, replayed between eager calls with other rows and slots."""
    from respect_amd.decoding.paged_kv import PagedKVCache
    c = PagedKVCache(2, 2, 64, pages=8, page=16, dtype=fmt)
    x, slots = torch.randn(9, 2, 64, device="cuda").to(BF), _i32(list(range(9)))
    c.write(0, x, x, slots)
    torch.cuda.synchronize()
    graphs = []
    for layer in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.write(layer, x, x, slots)
            out = c.read(layer, slots)
        graphs.append((g, out))
    for step in range(4):
        x.copy_(torch.randn(9, 2, 64, device="cuda") * 10.0 ** step)
        slots.copy_(_i32([(31 * i + step) % 128 for i in range(9)]))
        for g, _ in graphs:
            g.replay()
        want = values(*quantise(x.cpu(), fmt), fmt)
        for layer, (_, out) in enumerate(graphs):
            assert _same(out[0], want) and _same(out[1], want)
            assert _same(c.read(layer, slots)[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,D", [("mxfp8", 32), ("mxfp4", 32), ("mxfp8", 64), ("mxfp4", 128), ("mxfp4", 96), ("mxfp8", 256)])
def test_moved_rows(fmt, D):
    """Random runs of add, extend, fork, compact and free against plain rows, long lists among them."""
    from respect_amd.decoding.paged_kv import PagedKVCache
    rng = random.Random(D)
    g = torch.Generator().manual_seed(D)
    page, HK, layers = 16, 2, 2
    c = PagedKVCache(layers, HK, D, pages=200, page=page, sequences=24, dtype=fmt)
    rows = {}

    def fill(seqs, first, count):
        new = [torch.randn(layers, 2, n, HK, D, generator=g).to(BF) for n in count]
        slots = c.slots(seqs, first, count)
        for i in range(layers if new else 0):
            k, v = (torch.cat([x[i, j] for x in new]).cuda() for j in (0, 1))
            c.write(i, k, v, slots)
        return new
    for step in range(30):
        live = sorted(rows)
        some = rng.sample(live, rng.randint(0, len(live)))
        what = rng.choice(["add", "extend", "fork", "compact", "compact", "free"])
        print(step, what, len(some), flush=True)
        try:
            if what == "add":
                n = [rng.randint(0, 90) for _ in range(2)]
                seqs = c.add(n)
                rows.update(zip(seqs, fill(seqs, 0, n)))
            elif what == "extend":
                n, first = [rng.randint(0, 40) for _ in some], [c.length(s) for s in some]
                c.extend(some, n)
                for s, x in zip(some, fill(some, first, n)):
                    rows[s] = torch.cat((rows[s], x), 2)
            elif what == "fork" and some:
                for i, s in enumerate(c.fork(some[:2], 2)):
                    rows[s] = rows[some[:2][i // 2]].clone()
            elif what == "compact":
                starts = [rng.randint(0, c.length(s)) for s in some]
                paths = [sorted(rng.sample(range(c.length(s) - a), rng.randint(0, c.length(s) - a))) for s, a in zip(some, starts)]
                c.compact(some, starts, paths)
                for s, a, p in zip(some, starts, paths):
                    rows[s] = rows[s][:, :, [*range(a), *(a + i for i in p)]]
            elif what == "free":
                c.free(some[:1])
                for s in some[:1]:
                    del rows[s]
        except RuntimeError:
            pass                                                       # full
        for s, x in rows.items():
            slots = c.slots([s], 0, c.length(s))
            want = values(*quantise(x, fmt), fmt)
            for i in range(layers):
                for y, w in zip(c.read(i, slots), want[i]):
                    assert torch.equal(y.cpu().double(), w), (s, i)


@pytest.mark.gpu
def test_gpu_refusals_and_the_wrappers_own_path(monkeypatch):
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache
    from respect_amd.kernels.mx import MXRows, read_rows, write_rows
    p = MXRows.empty(2, 8, 64, "mxfp8")
    x, s = torch.randn(3, 2, 64, device="cuda").to(BF), _i32([1, 2, 5])
    for err, args in ((TypeError, (x.float(), x, p, p, s)), (RuntimeError, (x.cpu(), x, p, p, s)), (RuntimeError, (x, x, p, p, s.cpu())),
                      (ValueError, (x, x, p, MXRows.empty(2, 8, 64, "mxfp4"), s))):
        with pytest.raises(err):
            write_rows(*args)
    bf = torch.zeros(2, 8, 64, dtype=BF, device="cuda")
    for err, args in ((ValueError, (p, bf, s)), (ValueError, (bf, p, s)), (ValueError, (bf.transpose(1, 2), bf.transpose(1, 2), s)),
                      (RuntimeError, (bf, bf, s.cpu())), (TypeError, (bf, bf, s.long())), (ValueError, (bf, bf[:, :4], s))):
        with pytest.raises(err):
            read_rows(*args)

    class Leave:
        def __getattr__(self, name):
            return lambda *a: None

    def play(fmt):
        c = PagedKVCache(2, 2, 64, pages=30, page=4, sequences=9, dtype=fmt)
        g = torch.Generator(device="cuda").manual_seed(0)
        seqs = c.add([9, 4, 13])
        x = torch.randn(26, 2, 64, generator=g, device="cuda").to(BF)
        for layer in range(2):
            c.write(layer, x, -x, c.slots(seqs, 0, [9, 4, 13]))
        out = [c.fork(seqs, 2)]
        c.extend(out[0][:2], [3, 1])
        c.compact(seqs, [1, 0, 6], [[0, 2, 5], [], [3, 4]])
        table, lens = c.tables(seqs + out[0])
        out += [table.tolist(), lens.tolist(), c.free_pages, c._t.shared(out[0], 1)]
        got = [c.read(layer, c.slots(seqs + out[0], 0, lens.tolist())) for layer in range(2)]
        return out, [t for kv in got for t in kv]
    for fmt in ("bf16", "mxfp8", "mxfp4"):
        a, ta = play(fmt)
        with monkeypatch.context() as m:
            m.setattr(_lib, "_calls", Leave())
            b, tb = play(fmt)
        # rows that extend made room for hold what was there before: equal runs, equal rows
        assert a == b and all(_same(y, z) for y, z in zip(ta, tb))
