"""Attention over caches of 8 and 4 bits and over beginnings that sequences share
(kernels.paged_attention) against 64-bit attention over the values that the codes stand for:
formats, head layouts, pages, lengths at and below the shared keys, bad pages; a sequence's bits do
not depend on who shares its beginning; captured calls; plans and refusals on the CPU."""
import random

import pytest
import torch

from _mx import quantise, values

BF = torch.bfloat16
FORMATS = ["bf16", "mxfp8", "mxfp4"]
HEADS = [(32, 8, 128), (8, 2, 64), (16, 1, 128), (3, 1, 32), (4, 2, 256), (5, 5, 64)]


def _lib():
    from respect_amd import _lib as L
    if not L.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    return L


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _q(B, H, D, seed=1):
    return torch.randn(B, H, D, generator=torch.Generator().manual_seed(seed)).to(BF)


def _cache(lens, page, HK, D, fmt, members=(), keys=(), seed=0, spare=3):
    """(kc, vc as the call takes them, table, [(k, v) float64 per sequence]): scattered pages, a
    group's full pages of shared keys held together, everything no sequence holds NaN."""
    from respect_amd.kernels.mx import MXRows
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    common = [k // page for m, k in zip(members, keys) for _ in range(m)] or [0] * len(lens)
    common = [min(c, u) for c, u in zip(common, used)]
    pages = sum(used) + spare + sum(k // page for k in keys)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), max(used + [1])), -7, dtype=torch.int32)
    b = at = 0
    for m, k in zip(members, keys):
        for i in range(m):
            n = common[b + i] if i else min(k // page, table.shape[1])   # the first one's row names them all
            table[b + i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        b, at = b + m, at + k // page
    for i, n in enumerate(used):
        if n > common[i]:
            table[i, common[i]:n] = torch.tensor(order[at:at + n - common[i]], dtype=torch.int32)
            at += n - common[i]
    # Random keys everywhere, then NaN where nobody looks.
    kv = [torch.randn(HK, pages * page, D, generator=g).to(BF) for _ in range(2)]
    held = torch.zeros(pages * page, dtype=torch.bool)
    rows = []
    for b, n in enumerate(lens):
        j = torch.arange(max(n, 0))
        rows.append(table[b, j // page].long() * page + j % page)
        held[rows[-1]] = True
    b = 0
    for m, k in zip(members, keys):
        if m and k:
            held.view(pages, page)[table[b, :min(k // page, table.shape[1])].long()] = True
        b += m
    for x in kv:
        x[:, ~held] = float("nan")
    if fmt == "bf16":
        pools, real = [x.cuda() for x in kv], [x.double() for x in kv]
    else:
        coded = [quantise(x, fmt) for x in kv]
        pools = [MXRows(c.cuda(), s.cuda(), fmt) for c, s in coded]
        real = [values(c, s, fmt) for c, s in coded]
    return *pools, table, [tuple(x[:, r] for x in real) for r in rows]


def _exact(q, rows, shared=False, scale=None):
    """(result, bound) in float64.  As in test_paged_attention: p as two bf16 terms, off by 2^-15 p,
    fp32 sums and scores, one rounding of the result.  Shared keys: p rounded to bf16, off by
    2^-8 p at most, in the product and in the sum alike: numerator and denominator move by 2^-8
    of themselves, and their quotient by (a + |o|) 2^-8 / (1 - 2^-8), a = sum p |v|."""
    B, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b, (k, v) in enumerate(rows):
        n = k.shape[1]
        for h in range(H if n else 0):
            kd, vd, qd = k[h // (H // k.shape[0])], v[h // (H // k.shape[0])], q[b, h].double()
            p = torch.softmax(kd @ qd * scale, 0)
            o, a = p @ vd, p @ vd.abs()
            es = 2.0 ** -24 * ((D + 8) * float((kd.abs() @ qd.abs()).max()) * scale + 8)
            out[b, h] = o
            bound[b, h] = (a * (2.0 ** -15 + 2 * es + 2 * (n + 64) * 2.0 ** -24) + o.abs() * 2.0 ** -8) * 1.02
            if shared:
                bound[b, h] += (a + o.abs()) * 2.0 ** -8 * 1.01
    return out, bound


def _check(got, want, bound):
    assert torch.isfinite(got.float()).all()
    worst = float(((got.double().cpu() - want).abs() / (bound + 1e-30)).max())
    print(f"max err / bound {worst:.3f}", flush=True)
    assert worst <= 1


def _bits_equal(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def _plan(members, keys, group, **kw):
    from respect_amd.kernels.paged_attention import SharedPrefix
    return SharedPrefix(members, keys, group, **kw)


# ------------------------------------------------------------------ on the CPU

def test_plans():
    _lib()
    p = _plan([1, 3, 0, 2, 40], [500, 130, 900, 63, 1000], 4, device="cpu")
    assert p.B == 46 and p.longest == 960
    assert p.prefix.tolist() == [0] + [128] * 3 + [0] * 2 + [960] * 40
    t = p.tiles.tolist()
    assert t[0] == [1, 12, 0, 0, 1, 128, 0, 0] and t[1] == [6, 128, 0, 0, 1, 960, 0, 0] and t[5] == [6, 32, 128, 0, 4, 960, 0, 0]
    for keys in (64, 128, 192, 4095, 4096, 4160, 8000, 16384, 16448, 32768, 32832, 131072, 1 << 30, (1 << 31) - 1):
        for members, group in ((2, 1), (8, 4), (9, 4), (20, 4), (33, 4), (97, 4), (70, 16)):
            taken = {}
            for b0, rows, row0, split, splits, n, _, _ in _plan([members], [keys], group, device="cpu").tiles.tolist():
                assert b0 == 0 and n == keys // 64 * 64 and row0 % 128 == 0 and rows == min(128, members * group - row0)
                assert 1 <= splits <= (4 if rows <= 32 else 2 if rows <= 64 else 1)
                taken.setdefault(row0, []).extend(range(split, split + splits))
            assert sorted(taken) == list(range(0, members * group, 128))
            assert all(sorted(x) == list(range(len(x))) == list(range(len(taken[0]))) for x in taken.values())
            assert len(taken[0]) <= 64 and 128 * len(taken[0]) < keys // 64 * 64 + 128
    e = _plan([], [], 4, device="cpu")
    assert e.B == 0 and e.longest == 0 and len(e.tiles) == 0
    for bad in (([1], [1, 2], 4), ([-1], [5], 4), ([2], [-5], 4), ([2], [5], 0), ([2], [5], 17), ([1 << 28], [64], 16),
                ([2], [1 << 31], 4)):
        with pytest.raises(ValueError):
            _plan(*bad, device="cpu")
    for bad in (([1.5], [64], 4), ([2], [64.0], 4), ([2], [64], 4.0)):
        with pytest.raises(TypeError):
            _plan(*bad, device="cpu")


def test_groups_of_a_cache():
    """Groups by the full pages that neighbours begin with, cut so that most keys are shared."""
    _lib()
    from respect_amd.decoding.paged_kv import PagedKVCache, PageTable
    t = PageTable(100, 4, 64)
    a, b, c = t.add([17, 40, 8])
    fa, fb = t.fork([a], 3), t.fork([b], 2)
    assert t.shared([a, *fa, b, *fb, c], 1) == ([4, 3, 1], [16, 40, 0])
    assert t.shared([a, b, fa[0], fb[0]], 1) == ([1] * 4, [0] * 4)
    assert t.shared([a, *fa, b, *fb], 17) == ([1] * 4 + [3], [0] * 4 + [40])
    assert t.shared([], 1) == ([], []) and t.shared([c], 1) == ([1], [0])
    assert t.shared([a, a], 1) == ([2], [16])                 # the same one twice
    # a fork cut back shares what is left; one compacted into shared pages leaves them
    t.compact(fb[:1], 10, [[]])
    assert t.shared([b, *fb], 1) == ([3], [8]) and t.shared([fb[1], b, fb[0]], 1) == ([2, 1], [40, 0])
    t.compact([fa[0]], 0, [[1, 2, 3, 4, 5]])
    assert t.shared([a, fa[0]], 1) == ([1, 1], [0, 0])
    # a common beginning of all against longer ones of some
    t2 = PageTable(400, 4, 64)
    root, = t2.add([8])
    kids = t2.fork([root], 2)
    t2.extend(kids, 80)
    g0, g1 = t2.fork([kids[0]], 3), t2.fork([kids[1]], 3)
    assert t2.shared(g0 + g1, 1) == ([3, 3], [88, 88])
    with pytest.raises(ValueError):
        t2.shared([99], 1)
    cache = PagedKVCache(1, 2, 64, pages=64, page=16, device="cpu")
    s, = cache.add([300])
    seqs = cache._t.fork([s], 2)                              # no rows move on the CPU
    p = cache.shared([s, *seqs], 8)
    assert (p.members, p.group, p.prefix.tolist()) == ([3], 4, [256] * 3)
    assert cache.shared([s, *seqs], 8, least=289).longest == 0
    for heads in (0, 3, -2):
        with pytest.raises(ValueError):
            cache.shared(seqs, heads)
    rng = random.Random(5)
    for _ in range(60):                                       # the cut against all cuts
        t = PageTable(500, 2, 64)
        seqs = t.add([rng.randint(0, 12) for _ in range(2)])
        for _ in range(6):
            s = t.fork([rng.choice(seqs)], 1)
            t.extend(s, rng.randint(0, 6))
            seqs += s
        batch = [rng.choice(seqs) for _ in range(rng.randint(1, 7))]
        tables = [t.table([s])[0][0][:t.length(s) // 2].tolist() for s in batch]

        def common(lo, hi):
            n = 0
            while all(len(x) > n and x[n] == tables[lo][n] for x in tables[lo:hi]):
                n += 1
            return 2 * n

        def best(lo):
            if lo == len(batch):
                return 0
            return max(best(hi) + (hi - lo - 1) * (common(lo, hi) if hi - lo > 1 else 0) for hi in range(lo + 1, len(batch) + 1))
        members, keys = t.shared(batch, 1)
        assert sum(members) == len(batch)
        at = 0
        for m, k in zip(members, keys):
            assert k == (common(at, at + m) if m > 1 else 0)
            at += m
        assert sum((m - 1) * k for m, k in zip(members, keys)) == best(0)


def test_refusals():
    L = _lib()
    from respect_amd.kernels.mx import MXRows
    from respect_amd.kernels.paged_attention import paged_attn
    q, table, lens = _q(2, 4, 64), torch.zeros(2, 8, dtype=torch.int32), torch.tensor([5, 6], dtype=torch.int32)
    bf = torch.zeros(2, 64, 64, dtype=BF)
    p8, p4 = (MXRows.empty(2, 64, 64, f, device="cpu") for f in ("mxfp8", "mxfp4"))
    for args in ((q, p8, p4, table, lens, 16), (q, p8, bf, table, lens, 16), (q, bf, p8, table, lens, 16),
                 (_q(2, 4, 128), p8, p8, table, lens, 16), (q, p8, p8, table, lens, 48), (q, p8, p8, table[0], lens, 16)):
        with pytest.raises(ValueError):
            paged_attn(*args)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_attn(q, p8, p8, table, lens, 16)
    lib = L.lib()

    def call(shared, B=2, H=4, HK=2, D=64, pages=4, page=16, width=8, scale=0.1, fmt=8, p=16, s=1, st=64, ws=1 << 20, table=16, lens=16,
             prefix=16, tiles=16, n=1, longest=64):
        a = (p, 256, 64, p, 4096, st, s, 128, 2, p, 4096, st, s, 128, 2, table, 8, lens)
        b = (p, 256, 64, B, H, HK, D, pages, page, width, scale, fmt, 16, ws, None)
        return lib.rspx_paged_attn_shared(*a, prefix, tiles, n, longest, *b) if shared else lib.rspx_paged_attn_mx(*a, *b)
    for sh in (False, True):
        assert call(sh, H=3) == -1 and call(sh, B=-1) == -1 and call(sh, pages=0) == -1 and call(sh, page=12) == -1
        assert call(sh, width=-1) == -1 and call(sh, scale=0.0) == -1 and call(sh, p=0) == -1 and call(sh, lens=0) == -1
        assert call(sh, table=0) == -1 and call(sh, s=0) == -1 and call(sh, pages=1 << 28) == -1
        assert call(sh, D=96) == -2 and call(sh, H=34) == -2 and call(sh, fmt=6) == -2
        assert call(sh, p=8) == -4 and call(sh, st=72) == -4 and call(sh, st=1 << 31) == -2 and call(sh, st=-64) == -1
        assert call(sh, width=1024, ws=16) == -3
        assert call(sh, B=0) == 0
    assert call(False, fmt=16) == -2
    assert call(True, prefix=0) == -1 and call(True, tiles=0) == -1 and call(True, n=-1) == -1 and call(True, longest=-1) == -1
    assert call(True, longest=129) == -1 and call(True, n=1 << 23) == -2 and call(True, ws=16) == -3
    assert lib.rspx_paged_attn_shared_workspace_bytes(2, 4, 64, 16, 8, 0, 16) == 0
    assert lib.rspx_paged_attn_shared_workspace_bytes(2, 4, 64, 16, 8, 64, 8) == 2 * 4 * 2 * 66 * 4
    assert lib.rspx_paged_attn_shared_workspace_bytes(2, 4, 96, 16, 8, 64, 4) == -1
    assert lib.rspx_paged_attn_shared_workspace_bytes(2, 4, 64, 16, 8, 64, 5) == -1
    assert lib.rspx_shared_plan(None, None, 1, 4, None, None) == -1 and lib.rspx_shared_plan(None, None, 0, 4, None, None) == 0


# ------------------------------------------------------------------ caches of 8 and 4 bits

@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS[1:])
@pytest.mark.parametrize("H,HK,D", HEADS)
@pytest.mark.parametrize("page", [1, 16, 256])
def test_mx_against_64_bits(fmt, H, HK, D, page):
    from respect_amd.kernels.paged_attention import paged_attn
    lens = [1, 0, 31, 32, 33, 127, 128, 129, 255, 257, 600]
    kc, vc, table, rows = _cache(lens, page, HK, D, fmt, seed=H + page)
    q = _q(len(lens), H, D)
    got = paged_attn(q.cuda(), kc, vc, table.cuda(), _i32(lens), page)
    _check(got, *_exact(q, rows))
    assert (got[1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS[1:])
def test_mx_longer_than_the_shortest_splits(fmt):
    from respect_amd.kernels.paged_attention import paged_attn
    lens = [511, 512, 513, 4097, 8191, 8192, 8193, 20001]
    kc, vc, table, rows = _cache(lens, 32, 1, 64, fmt, seed=4)
    q = _q(len(lens), 4, 64)
    _check(paged_attn(q.cuda(), kc, vc, table.cuda(), _i32(lens), 32, sm_scale=0.3), *_exact(q, rows, scale=0.3))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS[1:])
def test_mx_equals_bf16_rows_of_the_same_values(fmt):
    """The products see the codes' values exactly: alike in order where head_dim's is (32), and to
    rounding elsewhere; a sequence alone or in a batch, other pages and strides: the same bits."""
    from respect_amd.kernels.mx import MXRows, read_rows
    from respect_amd.kernels.paged_attention import paged_attn
    for D in (32, 128):
        lens = [700, 45, 1300, 256]
        kc, vc, table, rows = _cache(lens, 16, 2, D, fmt, seed=2)
        q = _q(4, 8, D).cuda()
        all_ = paged_attn(q, kc, vc, table.cuda(), _i32(lens), 16)
        kb, vb = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in
                  read_rows(kc, vc, torch.arange(kc.shape[1], dtype=torch.int32, device="cuda")))
        bf = paged_attn(q, kb.transpose(0, 1), vb.transpose(0, 1), table.cuda(), _i32(lens), 16)
        if D == 32:
            assert torch.equal(bf, all_)
        _check(bf, *_exact(q.cpu(), rows))
        for b, n in enumerate(lens):
            assert torch.equal(paged_attn(q[b:b + 1], kc, vc, table[b:b + 1].cuda(), _i32([n]), 16)[0], all_[b])
        # slot-major pools with a pitch, out with one
        def pitched(p):
            c, s = (torch.zeros(p.shape[1], 2, t.shape[2] + w, dtype=torch.uint8, device="cuda") for t, w in ((p.codes, 16), (p.scales, 1)))
            c[..., :p.codes.shape[2]], s[..., 1:] = p.codes.transpose(0, 1), p.scales.transpose(0, 1)
            return MXRows(c.transpose(0, 1)[..., :p.codes.shape[2]], s.transpose(0, 1)[..., 1:], fmt)
        out = torch.zeros(4, 8, 2 * D, dtype=BF, device="cuda")
        paged_attn(q, pitched(kc), pitched(vc), table.cuda(), _i32(lens), 16, out=out[..., :D])
        assert torch.equal(out[..., :D], all_) and (out[..., D:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS[1:])
def test_mx_bad_pages_lengths_and_nan(fmt):
    from respect_amd.kernels.paged_attention import paged_attn
    lens, page = [300, 20, 20, 300, 300, 40], 16
    kc, vc, table, rows = _cache(lens, page, 2, 64, fmt, seed=3)
    q = _q(6, 4, 64)
    table[0, 18], table[3, 0], table[4, 19:] = kc.shape[1] // page, -1, 10 ** 9
    slot = int(table[5, 1]) * page + 3
    vc.scales[1, slot, 1] = 255                       # 32 values of one head are NaN
    got = paged_attn(q.cuda(), kc, vc, table.cuda(), _i32([300, -1, 16 * table.shape[1] + 1, 300, 300, 40]), page)
    assert torch.isnan(got[:4].float()).all()
    want, bound = _exact(q, rows)
    _check(got[4:5], want[4:5], bound[4:5])
    assert got[5, 2:, 32:].isnan().all()
    _check(got[5:, :2], want[5:, :2], bound[5:, :2])
    _check(got[5:, :, :32], want[5:, :, :32], bound[5:, :, :32])


# ------------------------------------------------------------------ shared beginnings

MEMBERS, KEYS = [1, 2, 3, 1, 40, 9], [300, 64, 100, 0, 640, 1024]


def _lens(page, seed):
    """Tails from none on, a few sequences shorter than their group's shared keys."""
    rng = random.Random(seed)
    lens = []
    for m, k in zip(MEMBERS, KEYS):
        k = k // page * page if page <= 64 else 0
        lens += [k + rng.choice([0, 1, 5, 31, 64, 100, 300]) for _ in range(m)]
    lens[4], lens[9], lens[12], lens[-1] = 20, 0, 639, 1
    return lens


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,HK,D", HEADS)
@pytest.mark.parametrize("page", [4, 64])
def test_shared_against_64_bits(fmt, H, HK, D, page):
    from respect_amd.kernels.paged_attention import paged_attn
    lens = _lens(page, H)
    keys = [k // page * page for k in KEYS]
    kc, vc, table, rows = _cache(lens, page, HK, D, fmt, MEMBERS, keys, seed=H + page)
    q = _q(len(lens), H, D)
    got = paged_attn(q.cuda(), kc, vc, table.cuda(), _i32(lens), page, shared=_plan(MEMBERS, keys, H // HK))
    _check(got, *_exact(q, rows, shared=True))
    assert (got[9] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_long_shared_keys(fmt):
    from respect_amd.kernels.paged_attention import paged_attn
    members, keys = [3, 2, 2, 2], [4096, 4160, 9984, 20032]
    lens = [4100, 4096, 4500, 4160, 4161, 10000, 9990, 20032, 21000]
    kc, vc, table, rows = _cache(lens, 64, 1, 64, fmt, members, keys, seed=5)
    q = _q(len(lens), 4, 64)
    plan = _plan(members, keys, 4)
    for scale in (None, 0.7):
        got = paged_attn(q.cuda(), kc, vc, table.cuda(), _i32(lens), 64, sm_scale=scale, shared=plan)
        _check(got, *_exact(q, rows, shared=True, scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_bits_do_not_depend_on_who_shares(fmt):
    """Two of a group, all of it in another order, another batch around it, other pages; a batch
    where nothing is shared has the bits of a call without a plan."""
    from respect_amd.kernels.paged_attention import paged_attn
    H, HK, D, page, k = 32, 2, 128, 16, 768
    members, lens = [24], [k + 13 * i for i in range(24)]
    kc, vc, table, _ = _cache(lens, page, HK, D, fmt, members, [k], seed=1)
    q, table = _q(24, H, D).cuda(), table.cuda()
    all_ = paged_attn(q, kc, vc, table, _i32(lens), page, shared=_plan(members, [k], 16))
    for pick in ([0, 1], [7, 3], [23, 0, 11, 12, 5], list(range(23, -1, -1))):
        n = [lens[i] for i in pick]
        got = paged_attn(q[pick], kc, vc, table[pick], _i32(n), page, shared=_plan([len(pick)], [k], 16))
        assert torch.equal(got, all_[pick])
    pick = [3, 4, 5, 9, 3, 4]
    got = paged_attn(q[pick], kc, vc, table[pick], _i32([lens[i] for i in pick]), page, shared=_plan([1, 2, 1, 2], [k] * 4, 16))
    assert torch.equal(got[[1, 2]], all_[[4, 5]]) and torch.equal(got[[4, 5]], all_[[3, 4]])
    alone = paged_attn(q, kc, vc, table, _i32(lens), page)
    assert torch.equal(got[[0, 3]], alone[[3, 9]])
    assert torch.equal(paged_attn(q, kc, vc, table, _i32(lens), page, shared=_plan([1] * 24, [k] * 24, 16)), alone)
    short = [min(n, 700) for n in lens]                          # all shorter than what they share
    assert torch.equal(paged_attn(q, kc, vc, table, _i32(short), page, shared=_plan(members, [k], 16)),
                       paged_attn(q, kc, vc, table, _i32(short), page))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("k", [64, 320, 832])
def test_any_number_of_members_gives_the_same_bits(fmt, D, k):
    """One to 136 rows a kv head, blocks of 32, 64 and 128 and what is left of them, splits that do
    not divide evenly among a workgroup's waves; own keys from none to more than a wave takes."""
    from respect_amd.kernels.paged_attention import paged_attn
    H, HK, page, B = 24, 3, 32, 17
    lens = [k + (0, 1, 32, 33, 7)[i % 5] for i in range(B)]
    kc, vc, table, rows = _cache(lens, page, HK, D, fmt, [B], [k], seed=D + k)
    q, table = _q(B, H, D).cuda(), table.cuda()
    all_ = paged_attn(q, kc, vc, table, _i32(lens), page, shared=_plan([B], [k], 8))
    _check(all_, *_exact(q.cpu(), rows, shared=True))
    for m in (2, 4, 5, 8, 9, 12, 16):
        got = paged_attn(q[-m:], kc, vc, table[-m:], _i32(lens[-m:]), page, shared=_plan([m], [k], 8))
        assert torch.equal(got, all_[-m:])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_bad_pages_among_the_shared(fmt):
    """A page that is none: NaN for all who read it, through the group or alone; bad lengths; the
    others keep their bits."""
    from respect_amd.kernels.paged_attention import paged_attn
    members, keys, page = [3, 3], [256, 512], 64
    lens = [300, 270, 100, 512, 600, 700]
    kc, vc, table, rows = _cache(lens, page, 2, 64, fmt, members, keys, seed=8)
    q, plan = _q(6, 8, 64), _plan(members, keys, 4)
    pages = kc.shape[1] // page
    good = paged_attn(q.cuda(), kc, vc, table.cuda(), _i32(lens), page, shared=plan)
    _check(good, *_exact(q, rows, shared=True))
    for bad in (pages, -1, 10 ** 9, -2 ** 31):
        t = table.clone()
        t[0, 3] = bad
        got = paged_attn(q.cuda(), kc, vc, t.cuda(), _i32(lens), page, shared=plan)
        assert got[:2].isnan().all() and torch.equal(got[2:], good[2:])
    got = paged_attn(q.cuda(), kc, vc, table.cuda(), _i32([300, -1, 0, 1 << 30, 600, 700]), page, shared=plan)
    assert got[[1, 3]].isnan().all() and (got[2] == 0).all() and torch.equal(got[[0, 4, 5]], good[[0, 4, 5]])


@pytest.mark.gpu
def test_infinite_values():
    """An infinite value reaches those who see it alone, and spoils no one else's."""
    from respect_amd.kernels.paged_attention import paged_attn
    members, keys, page = [3], [128], 16
    lens = [128, 140, 50]
    kc, vc, table, _ = _cache(lens, page, 1, 64, "bf16", members, keys)
    vc[0, int(table[0, 5]) * page + 4, 3] = float("inf")          # key 84
    got = paged_attn(_q(3, 4, 64).cuda(), kc, vc, table.cuda(), _i32(lens), page, shared=_plan(members, keys, 4))
    assert (got[:2, :, 3] == float("inf")).all() and torch.isfinite(got[:2, :, 4:]).all() and torch.isfinite(got[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_graphs_follow_tables_and_lengths(fmt):
    """Two captured calls, replayed in turn and at once on two streams, between eager ones, each with
    changed lengths."""
    from respect_amd.kernels.paged_attention import paged_attn
    members, keys, page = [4, 1, 3], [512, 0, 256], 16
    lens = [1300, 512, 700, 513, 5, 300, 256, 400]
    kc, vc, table, _ = _cache(lens, page, 2, 128, fmt, members, keys, seed=7)
    table, q, n, plan = table.cuda().clamp_(min=0), _q(8, 8, 128).cuda(), _i32(lens), _plan(members, keys, 4)
    paged_attn(q, kc, vc, table, n, page, shared=plan)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_attn(q, kc, vc, table, n, page, shared=plan)
            alone = paged_attn(q, kc, vc, table, n, page)
        graphs.append((g, out, alone))
    side = torch.cuda.Stream()
    for new in (lens, [512] * 4 + [1, 256, 255, 0], [600, 1, 2, 3, 4, 257, 258, 300], [x - 1 for x in lens]):
        n.copy_(_i32(new))
        graphs[0][0].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        eager, plain = paged_attn(q, kc, vc, table, n, page, shared=plan), paged_attn(q, kc, vc, table, n, page)
        torch.cuda.current_stream().wait_stream(side)
        # Sequence 6 reads past its pages in one of them, rows that may be NaN: bits are compared.
        for _, out, alone in graphs:
            assert _bits_equal(out, eager) and _bits_equal(alone, plain)
            for x in (out, alone):
                assert torch.isfinite(x[[0, 1, 2, 3, 4, 5, 7]].float()).all()
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_more_sequences_than_a_launch_takes():
    """2060 sequences, launched 1024 at a time, in groups that lie across the borders."""
    from respect_amd.kernels.paged_attention import paged_attn
    members, keys, page = [1000, 100, 900, 60], [128, 256, 64, 320], 16
    B = sum(members)
    lens = [k + 1 + (7 * b) % 30 for m, k in zip(members, keys) for b in range(m)]
    kc, vc, table, rows = _cache(lens, page, 2, 64, "mxfp8", members, keys, seed=B)
    q = _q(B, 4, 64)
    got = paged_attn(q.cuda(), kc, vc, table.cuda(), _i32(lens), page, shared=_plan(members, keys, 2))
    some = [0, 1, 999, 1000, 1023, 1024, 1025, 1099, 1100, 1999, 2000, 2047, 2048, 2059]
    _check(got[some], *_exact(q[some], [rows[b] for b in some], shared=True))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
def test_offsets_past_32_bits(fmt):
    """Pools whose heads and rows lie more than 2^32 bytes apart."""
    from respect_amd.kernels.mx import MXRows
    from respect_amd.kernels.paged_attention import paged_attn
    members, keys, page, D = [3], [64], 64, 64
    lens = [64, 100, 90]
    kc, vc, table, rows = _cache(lens, page, 2, D, fmt, members, keys, seed=2)
    far, at = (lambda t: [255 - int(x) for x in t]), {}
    width = 9000 * 8 if fmt == "bf16" else 1 << 18
    base = torch.zeros(2, 256 * page, width, dtype=BF if fmt == "bf16" else torch.uint8, device="cuda")
    new = table.clone()
    new[table >= 0] = 255 - table[table >= 0]
    pages = kc.shape[1] // page

    def place(parts, offset):
        out = []
        for p in parts:
            x = base[:, :, offset:offset + p.shape[2]]
            x.view(2, 256, page, -1)[:, [255 - i for i in range(pages)]] = p.view(2, pages, page, -1)
            out.append(x)
            offset += 4096
        return out
    if fmt == "bf16":
        (k2,), (v2,) = place([kc], 0), place([vc], 32768)
    else:
        k2, v2 = MXRows(*place([kc.codes, kc.scales], 0), fmt), MXRows(*place([vc.codes, vc.scales], 32768), fmt)
    q = _q(3, 4, D)
    got = paged_attn(q.cuda(), k2, v2, new.cuda(), _i32(lens), page, shared=_plan(members, keys, 2))
    _check(got, *_exact(q, rows, shared=True))
    assert torch.equal(got, paged_attn(q.cuda(), kc, vc, table.cuda(), _i32(lens), page, shared=_plan(members, keys, 2)))


@pytest.mark.gpu
def test_gpu_refusals_and_the_wrappers_own_path(monkeypatch):
    from respect_amd import _lib
    from respect_amd.kernels.paged_attention import paged_attn

    class Leave:
        def __getattr__(self, name):
            return lambda *a: None
    members, keys, lens = [2, 1], [64, 0], [70, 64, 30]
    for fmt in FORMATS:
        kc, vc, table, _ = _cache(lens, 16, 2, 64, fmt, members, keys)
        q, table, n, plan = _q(3, 4, 64).cuda(), table.cuda(), _i32(lens), _plan(members, keys, 2)
        a = [paged_attn(q, kc, vc, table, n, 16, shared=p) for p in (plan, None)]
        with monkeypatch.context() as m:
            m.setattr(_lib, "_calls", Leave())
            b = [paged_attn(q, kc, vc, table, n, 16, shared=p) for p in (plan, None)]
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        out = torch.empty_like(q)
        assert torch.equal(paged_attn(q, kc, vc, table, n, 16, out=out, shared=plan), a[0])
        for err, args in ((ValueError, dict(shared=_plan([2], [64], 2))), (ValueError, dict(shared=_plan(members, keys, 4))),
                          (ValueError, dict(shared=_plan(members, [1024, 0], 2))),
                          (RuntimeError, dict(shared=_plan(members, keys, 2, device="cpu")))):
            with pytest.raises(err):
                paged_attn(q, kc, vc, table, n, 16, **args)
        with pytest.raises(RuntimeError):
            paged_attn(q, kc, vc, table.cpu(), n, 16, shared=plan)
        empty = paged_attn(q[:0], kc, vc, table[:0], n[:0], 16, shared=_plan([], [], 2))
        assert empty.shape == (0, 4, 64)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError):
            _plan(members, keys, 2)
