"""Attention of one new token per sequence over a paged cache (kernels.paged_attention)
against 64-bit attention: page sizes, lengths from nothing to several splits, grouped heads,
scattered and shared pages, rows past a sequence's end and pages past its table that hold
NaN, bad pages and lengths; a sequence's bits do not depend on the batch; refusals on the CPU."""
import pytest
import torch

BF = torch.bfloat16


def _cache(lens, page, HK, D, seed=0, spare=3, width=None):
    """(kc, vc, table, [(k, v) per sequence]): scattered pages, everything no sequence holds NaN."""
    g = torch.Generator()
    g.manual_seed(seed)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g).tolist()
    kc, vc = (torch.full((HK, pages * page, D), float("nan"), dtype=BF) for _ in range(2))
    table = torch.full((len(lens), max(used + [1]) if width is None else width), -7, dtype=torch.int32)
    rows, at = [], 0
    for b, n in enumerate(lens):
        table[b, :used[b]] = torch.tensor(order[at:at + used[b]], dtype=torch.int32)
        at += used[b]
        k, v = (torch.randn(HK, n, D, generator=g).to(BF) for _ in range(2))
        j = torch.arange(n)
        slots = table[b, j // page].long() * page + j % page
        kc[:, slots], vc[:, slots] = k, v
        rows.append((k, v))
    return kc, vc, table, rows


def _exact(q, rows, scale=None):
    """(result, bound) in float64.  p enters the product as two bf16 terms: cut to 8 bits, which
    leaves a rest below 2^-7 p, and that rest rounded, off by half a step, 2^-8 of it at most:
    2^-15 p.  Sums and scores as in fp32, the result rounded to bf16 once."""
    B, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b, (k, v) in enumerate(rows):
        n = k.shape[1]
        for h in range(H if n else 0):
            kd, vd, qd = k[h // (H // k.shape[0])].double(), v[h // (H // k.shape[0])].double(), q[b, h].double()
            p = torch.softmax(kd @ qd * scale, 0)
            o, a = p @ vd, p @ vd.abs()
            es = 2.0 ** -24 * ((D + 8) * float((kd.abs() @ qd.abs()).max()) * scale + 8)
            out[b, h] = o
            bound[b, h] = (a * (2.0 ** -15 + 2 * es + 2 * (n + 64) * 2.0 ** -24) + o.abs() * 2.0 ** -8) * 1.02
    return out, bound


def _check(got, want, bound):
    assert torch.isfinite(got.float()).all()
    worst = float(((got.double().cpu() - want).abs() / (bound + 1e-30)).max())
    print(f"max err / bound {worst:.3f}", flush=True)
    assert worst <= 1


def _q(B, H, D, seed=1):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(B, H, D, generator=g).to(BF)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_refusals():
    from respect_amd import _lib
    from respect_amd.kernels.paged_attention import paged_attn
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    kc, vc, table, _ = _cache([5], 16, 2, 64)
    q, lens = _q(1, 4, 64), torch.tensor([5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_attn(q, kc, vc, table, lens, 16)
    for args in ((q, kc[:, :-1], vc[:, :-1], table, lens, 16), (q, kc, vc[:, :16], table, lens, 16),
                 (q, kc, vc, table[0], lens, 16), (q, kc, vc, table, lens[:0], 16), (q, kc, vc, table, lens, 0)):
        with pytest.raises(ValueError):
            paged_attn(*args)
    with pytest.raises(TypeError):
        paged_attn(q, kc, vc, table.long(), lens, 16)
    L = _lib.lib()

    def call(B=1, H=4, HK=2, D=64, pages=4, page=16, width=4, scale=0.1, p=16, st=64, ws=1 << 20, table=16, lens=16):
        return L.rspx_paged_attn(p, 256, st, p, 4096, 64, p, 4096, 64, table, 4, lens, p, 256, 64, B, H, HK, D, pages,
                                 page, width, scale, 16, ws, None)
    assert call(H=3) == -1 and call(B=-1) == -1 and call(pages=0) == -1 and call(page=12) == -1 and call(width=-1) == -1
    assert call(scale=0.0) == -1 and call(scale=float("nan")) == -1 and call(p=0) == -1 and call(lens=0) == -1
    assert call(table=0) == -1 and call(pages=1 << 28) == -1 and call(width=1 << 28) == -1
    assert call(D=96) == -2 and call(H=34) == -2 and call(H=5000, HK=5000) == -2
    assert call(p=8) == -4 and call(st=100) == -4
    assert call(width=1024, ws=16) == -3
    assert call(B=0) == 0
    assert L.rspx_paged_attn_workspace_bytes(1, 4, 64, 16, 16) == 0     # one split
    assert L.rspx_paged_attn_workspace_bytes(1, 4, 64, 16, 17) > 0
    assert L.rspx_paged_attn_workspace_bytes(1, 4, 96, 16, 16) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("H,HK,D", [(32, 8, 128), (8, 2, 64), (16, 1, 128), (3, 1, 32), (4, 2, 256), (5, 5, 64)])
@pytest.mark.parametrize("page", [1, 16, 64, 256])
def test_against_64_bits(H, HK, D, page):
    from respect_amd.kernels.paged_attention import paged_attn
    lens = [1, 0, 31, 32, 33, 127, 128, 129, 255, 257, 600]
    kc, vc, table, rows = _cache(lens, page, HK, D, seed=H + page)
    q = _q(len(lens), H, D)
    got = paged_attn(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), _i32(lens), page)
    _check(got, *_exact(q, rows))
    assert (got[1] == 0).all()


@pytest.mark.gpu
def test_longer_than_the_shortest_splits():
    """Lengths around the places where splits are added and grow."""
    from respect_amd.kernels.paged_attention import paged_attn
    lens = [511, 512, 513, 4097, 8191, 8192, 8193, 9000, 20001]
    kc, vc, table, rows = _cache(lens, 32, 1, 64, seed=4)
    q = _q(len(lens), 4, 64)
    got = paged_attn(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), _i32(lens), 32)
    _check(got, *_exact(q, rows))


@pytest.mark.gpu
def test_large_scores_and_scale():
    from respect_amd.kernels.paged_attention import paged_attn
    lens = [900, 40]
    kc, vc, table, rows = _cache(lens, 16, 2, 128, seed=6)
    q = (_q(2, 8, 128).float() * 20).to(BF)
    got = paged_attn(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), _i32(lens), 16, sm_scale=0.3)
    _check(got, *_exact(q, rows, 0.3))


@pytest.mark.gpu
def test_bits_do_not_depend_on_the_batch_or_the_pages():
    """Alone, in a batch, with other pages, a wider table, shared pages, strided tensors."""
    from respect_amd.kernels.paged_attention import paged_attn
    lens, H, HK, D = [700, 45, 1300, 256], 8, 2, 128
    kc, vc, table, rows = _cache(lens, 16, HK, D, seed=2)
    q = _q(4, H, D).cuda()
    all_ = paged_attn(q, kc.cuda(), vc.cuda(), table.cuda(), _i32(lens), 16)
    for b, n in enumerate(lens):
        one = paged_attn(q[b:b + 1], kc.cuda(), vc.cuda(), table[b:b + 1].cuda(), _i32([n]), 16)
        assert torch.equal(one[0], all_[b])
        k, v = (torch.zeros(HK, 2048, D, dtype=BF, device="cuda") for _ in range(2))
        k[:, :n], v[:, :n] = rows[b][0].cuda(), rows[b][1].cuda()
        flat = paged_attn(q[b:b + 1], k, v, torch.arange(32, device="cuda", dtype=torch.int32)[None], _i32([n]), 64)
        assert torch.equal(flat[0], all_[b])
    twice = paged_attn(q[[0, 0]], kc.cuda(), vc.cuda(), table[:1].cuda().expand(2, -1), _i32([700, 700]), 16)
    assert torch.equal(twice[0], all_[0]) and torch.equal(twice[1], all_[0])
    # [slots, HK, D] pools, q inside a wider row, out with a pitch, a table inside a wider one.
    ks, vs = (t.cuda().transpose(0, 1).contiguous().transpose(0, 1) for t in (kc, vc))
    wide = torch.zeros(4, H + 2, D, dtype=BF, device="cuda")
    wide[:, 1:-1] = q
    out = torch.zeros(4, H, 2 * D, dtype=BF, device="cuda")
    tw = torch.zeros(4, table.shape[1] + 5, dtype=torch.int32, device="cuda")
    tw[:, :table.shape[1]] = table.cuda()
    got = paged_attn(wide[:, 1:-1], ks, vs, tw[:, :table.shape[1]], _i32(lens), 16, out=out[..., :D])
    assert torch.equal(got, all_) and (out[..., D:] == 0).all()


@pytest.mark.gpu
def test_bad_pages_and_lengths_give_nan_rows():
    from respect_amd.kernels.paged_attention import paged_attn
    lens, page, H, HK, D = [300, 20, 20, 300, 300], 16, 4, 2, 64
    kc, vc, table, rows = _cache(lens, page, HK, D, seed=3)
    q = _q(5, H, D)
    pages = kc.shape[1] // page
    table[0, 18] = pages            # one past the pool
    table[3, 0] = -1
    table[4, 19:] = 10 ** 9         # behind the end: not read
    got = paged_attn(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), _i32([300, -1, 16 * table.shape[1] + 1, 300, 300]), page)
    assert torch.isnan(got[:4].float()).all()
    want, bound = _exact(q, rows)
    _check(got[4:], want[4:], bound[4:])


@pytest.mark.gpu
def test_infinite_values_at_the_end():
    """The last key's value is infinite: the columns are, the rest is finite."""
    from respect_amd.kernels.paged_attention import paged_attn
    kc, vc, table, _ = _cache([37], 16, 1, 64)
    slot = int(table[0, 2]) * 16 + 4
    vc[0, slot, 3] = float("inf")
    got = paged_attn(_q(1, 4, 64).cuda(), kc.cuda(), vc.cuda(), table.cuda(), _i32([37]), 16)
    assert (got[..., 3] == float("inf")).all() and torch.isfinite(got[..., 4:]).all() and torch.isfinite(got[..., :3]).all()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pools whose heads and rows lie more than 2^32 bytes apart."""
    from respect_amd.kernels.paged_attention import paged_attn
    n, page, D = 200, 64, 64
    base = torch.zeros(2, 256 * 64, 9000 * 8, dtype=BF, device="cuda")   # 4.7 GB
    kc = base[:, :, :D]
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    table = _i32([[255, 3, 254, 128]])
    j = torch.arange(n, device="cuda")
    slots = table[0, j // page].long() * page + j % page
    k, v = (torch.randn(2, n, D, generator=g, device="cuda").to(BF) for _ in range(2))
    vc = base[:, :, 4096:4096 + D]
    kc[:, slots], vc[:, slots] = k, v
    q = _q(1, 4, D)
    got = paged_attn(q.cuda(), kc, vc, table, _i32([n]), page)
    _check(got, *_exact(q, [(k.cpu(), v.cpu())]))


@pytest.mark.gpu
def test_graph_follows_tables_and_lengths():
    """Two captured calls, replayed in turn and at once on two streams, between eager ones, each
    with changed tables and lengths."""
    from respect_amd.kernels.paged_attention import paged_attn
    lens = [1300, 5, 700]
    kc, vc, table, _ = _cache(lens, 16, 2, 128, seed=7)
    kc, vc, table, q = kc.cuda(), vc.cuda(), table.cuda(), _q(3, 8, 128).cuda()
    table.clamp_(min=0)
    n = _i32(lens)
    paged_attn(q, kc, vc, table, n, 16)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_attn(q, kc, vc, table, n, 16)
        graphs.append((g, out))
    side = torch.cuda.Stream()
    for step, new in enumerate(([1300, 5, 700], [257, 0, 699], [1, 2, 3], [1299, 4, 650])):
        n.copy_(_i32(new))
        graphs[0][0].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        eager = paged_attn(q, kc, vc, table, n, 16)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(graphs[0][1], eager) and torch.equal(graphs[1][1], eager)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_gpu_refusals_and_empty():
    from respect_amd.kernels.paged_attention import paged_attn
    kc, vc, table, _ = _cache([5], 16, 2, 64)
    kc, vc, table, q, n = kc.cuda(), vc.cuda(), table.cuda(), _q(1, 4, 64).cuda(), _i32([5])
    with pytest.raises(TypeError):
        paged_attn(q.float(), kc, vc, table, n, 16)
    with pytest.raises(ValueError):
        paged_attn(q, kc.transpose(1, 2).contiguous().transpose(1, 2), vc, table, n, 16)
    with pytest.raises(RuntimeError):
        paged_attn(q, kc, vc, table.cpu(), n, 16)
    with pytest.raises(RuntimeError):
        paged_attn(q, kc[:, :48], vc[:, :48], table, n, 24)      # no power of two
    assert paged_attn(q[:0], kc, vc, table[:0], n[:0], 16).shape == (0, 4, 64)
    assert (paged_attn(q, kc, vc, table[:, :0], _i32([0]), 16) == 0).all()


@pytest.mark.gpu
def test_more_sequences_than_a_launch_takes():
    """1030 and 2060 sequences, launched 1024 at a time: rows on both sides of the borders against
    64 bits, every row the bits of the same sequence in a small batch."""
    from respect_amd.kernels.paged_attention import paged_attn
    H, HK, D, page = 4, 2, 64, 16
    for B in (1030, 2060):
        lens = [(7 * b) % 40 for b in range(B)]
        for b, n in ((0, 600), (1023, 700), (1024, 900), (1029, 513), (B - 2, 1300), (B - 1, 257)):
            lens[b] = n
        kc, vc, table, rows = _cache(lens, page, HK, D, seed=B)
        q, kc, vc, table = _q(B, H, D, seed=B).cuda(), kc.cuda(), vc.cuda(), table.cuda()
        got = paged_attn(q, kc, vc, table, _i32(lens), page)
        some = [0, 1, 1022, 1023, 1024, 1025, 1028, 1029, B - 3, B - 2, B - 1]
        _check(got[some], *_exact(q[some].cpu(), [rows[b] for b in some]))
        for a in range(0, B, 200):
            part = paged_attn(q[a:a + 200], kc, vc, table[a:a + 200], _i32(lens[a:a + 200]), page)
            assert torch.equal(part, got[a:a + 200]), a
