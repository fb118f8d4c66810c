"""Plans of shared beginnings in batches that change: sequences cut back below what they share, the
first of a group among them, and grown again."""
import pytest
import torch

from test_shared_attention import FORMATS, _cache, _check, _exact, _i32, _plan, _q

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,HK,D", [(32, 8, 128), (3, 3, 32), (8, 2, 64), (4, 2, 256)])
def test_any_of_a_group_may_be_short(fmt, H, HK, D):
    """Sequences cut back below the shared keys, whose table rows hold no page or other ones behind
    their ends: they are taken by themselves, the others keep their bits.  40 members with one head
    each to four: one tile, or a second one whose sequences are others."""
    from respect_amd.kernels.paged_attention import paged_attn
    page, k, B = 16, 256, 40
    full = [k + (0, 7, 40)[i % 3] for i in range(B)]
    kc, vc, table, rows = _cache(full, page, HK, D, fmt, [B], [k], seed=H)
    plan, q = _plan([B], [k], H // HK), _q(B, H, D).cuda()
    good = paged_attn(q, kc, vc, table.cuda(), _i32(full), page, shared=plan)
    _check(good, *_exact(q.cpu(), rows, shared=True))
    pages = kc.shape[1] // page
    for short in ([0], [0, 1, 2], list(range(34)), [0, 5, 33, 39], list(range(39)), list(range(B))):
        for behind in (-1, pages - 1):
            lens, t = list(full), table.clone()
            for b in short:
                lens[b] = (20, 255, 0, 33)[b % 4]
                t[b, -(-lens[b] // page):] = behind
            got = paged_attn(q, kc, vc, t.cuda(), _i32(lens), page, shared=plan)
            alone = paged_attn(q, kc, vc, t.cuda(), _i32(lens), page)
            long = [b for b in range(B) if b not in short]
            assert torch.equal(got[long], good[long]), (short, behind)
            assert torch.equal(got[short], alone[short]), (short, behind)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_first_fork_that_is_cut_back(fmt):
    """A cache's forks, the first one compacted below the shared keys, then trimmed or extended: the
    others have the bits of a plan of their own, it those of a call without one."""
    from respect_amd.decoding.paged_kv import PagedKVCache
    from respect_amd.kernels.paged_attention import paged_attn
    H, HK, D, page = 8, 2, 64, 16
    for again in ("trim", "extend"):
        cache = PagedKVCache(1, HK, D, pages=80, page=page, dtype=fmt)
        g = torch.Generator().manual_seed(1)
        for pool in (cache.k[0], cache.v[0]):                    # rows no sequence has yet are NaN or large
            if fmt == "bf16":
                pool.fill_(float("nan"))
            else:
                pool.scales.fill_(255)
        s, = cache.add([300])
        x = torch.randn(2, 300, HK, D, generator=g).to(BF).cuda()
        cache.write(0, *x, cache.slots([s], 0, 300))
        seqs = [s, *cache.fork([s], 2)]
        plan, others = cache.shared(seqs, H), cache.shared(seqs[1:], H)
        assert plan.longest == others.longest == 256
        cache.compact([s], 20, [[]])
        if again == "trim":
            cache.trim([s])
        else:
            cache.extend([s], 200)                               # pages of its own where it shared
            cache.write(0, *x[:, :200], cache.slots([s], 20, 200))
        q = _q(3, H, D).cuda()
        table, lens = cache.tables(seqs)
        got = paged_attn(q, cache.k[0], cache.v[0], table, lens, page, shared=plan)
        want = paged_attn(q[1:], cache.k[0], cache.v[0], table[1:], lens[1:], page, shared=others)
        assert torch.isfinite(got.float()).all() and torch.equal(got[1:], want)
        assert torch.equal(got[:1], paged_attn(q[:1], cache.k[0], cache.v[0], table[:1], lens[:1], page))
