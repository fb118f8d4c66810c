"""Plans of shared beginnings in batches that change: sequences cut back below what they share, the
first of a group among them, and grown again, freed, in another order; what refuses them."""
import numpy as np
import pytest
import torch

from test_shared_attention import FORMATS, _cache, _check, _exact, _i32, _plan, _q

BF = torch.bfloat16


def _forks():
    """A cache on the CPU with two documents and two forks of each, (cache, sequences, plan)."""
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    cache = PagedKVCache(1, 2, 64, pages=200, page=16, device="cpu")
    a, b = cache.add([300, 700])
    fa, fb = cache._t.fork([a], 2), cache._t.fork([b], 2)        # no rows move on the CPU
    seqs = [a, *fa, b, *fb]
    plan = cache.shared(seqs, 8)
    assert plan.members == [3, 3] and [x.tolist() for x in plan.groups] == [[3, 3], [256, 640]]
    assert cache.holds(seqs, plan)
    return cache, seqs, plan


def test_a_plan_holds_while_sequences_grow():
    cache, seqs, plan = _forks()
    # the longer ones share 256 keys too, the shorter ones have no 640 and are taken by themselves
    assert cache.holds([*seqs[3:], *seqs[:3]], plan)
    cache._t.extend(seqs, [1, 20, 500, 0, 5, 16])
    assert cache.holds(seqs, plan) and cache.holds([*seqs[3:], *seqs[:3]], plan)
    cache._t.extend(seqs[:1], 400)                               # two with 640 keys now, in pages of their own
    assert cache.holds(seqs, plan) and not cache.holds([*seqs[3:], *seqs[:3]], plan)
    assert cache.holds([seqs[i] for i in (2, 0, 1, 5, 4, 3)], plan)      # another order in which it is as right
    more = cache._t.fork(seqs, 1)
    assert cache.holds(more, plan) and cache.holds([*seqs[:3], *more[3:]], plan)
    alone = cache.shared(seqs[:1] + seqs[3:4], 8)
    assert alone.longest == 0 and cache.holds(seqs[2:4], alone)
    empty = cache.shared([], 8)
    assert cache.holds([], empty) and not cache.holds(seqs, empty) and not cache.holds([], plan)


def test_a_plan_of_other_sequences_does_not_hold():
    cache, seqs, plan = _forks()
    a, fa, ga, b, fb, gb = seqs
    for other in ([a, b, fa, fb, ga, gb], [a, fa, b, ga, fb, gb], seqs[:5], [*seqs, a], []):
        assert not cache.holds(other, plan)
    with pytest.raises(ValueError):
        cache.holds([*seqs[:5], 99], plan)
    new, = cache.add([700])                                      # as long, in pages of its own
    assert not cache.holds([a, fa, ga, b, fb, new], plan)
    cache._t.free([gb, new])
    with pytest.raises(ValueError):
        cache.holds(seqs, plan)                                  # freed
    took = cache.add([700, 20])
    assert gb in took                                            # its number, taken by another
    assert cache.holds(seqs, plan) is (cache.length(gb) < 640)
    cache._t.extend([gb], 700)
    assert not cache.holds(seqs, plan)


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("trim", [False, True])
def test_a_plan_and_sequences_that_are_cut_back(which, trim):
    """Cut back below the shared keys a sequence is by itself; as long again it has rows of its own."""
    cache, seqs, plan = _forks()
    P = (256, 640)[which // 3]
    s = seqs[which]
    cache._t.compact([s], P + 3, [[]])
    assert cache.holds(seqs, plan)
    cache._t.compact([s], 20, [[]])
    if trim:
        cache._t.trim([s])
    assert cache.holds(seqs, plan)
    cache._t.extend([s], P - 20 - 1)
    assert cache.holds(seqs, plan)
    cache._t.extend([s], 1)
    assert not cache.holds(seqs, plan)
    cache._t.undo()
    assert cache.holds(seqs, plan)
    cache._t.extend([s], 1)
    assert cache.shared(seqs, 8).members != plan.members or which in (1, 4)
    assert cache.holds(seqs, cache.shared(seqs, 8))


def test_alike_against_tables():
    """Random groups of random forks, compared with the sequences' tables."""
    import random
    from respect_amd.decoding.paged_kv import PageTable
    _forks()
    rng, seen = random.Random(3), set()
    for _ in range(300):
        t = PageTable(500, 4, 64)
        seqs = t.add([rng.randint(0, 40) for _ in range(2)])
        for _ in range(5):
            s = t.fork([rng.choice(seqs)], 1)
            if rng.random() < 0.4:
                t.compact(s, rng.randint(0, t.length(s[0])), [[]])
            t.extend(s, rng.randint(0, 12))
            seqs += s
        members = [rng.randint(0, 3) for _ in range(rng.randint(0, 4))]
        keys = [rng.randint(0, 30) for _ in members]
        batch = [rng.choice(seqs) for _ in range(sum(members))]
        want, at = True, 0
        for m, k in zip(members, keys):
            rows = {tuple(t.table([s])[0][0][:-(-k // 4)].tolist()) for s in batch[at:at + m] if t.length(s) >= k}
            want, at = want and len(rows) <= 1, at + m
        assert t.alike(batch, np.array(members, np.int64), np.array(keys, np.int64)) is want
        seen.add(want)
    assert seen == {True, False}
    for members, keys in (([-1], [4]), ([1], [-4]), ([2], [4])):
        y = t._lib.rspx_pages_alike(t.handle, t._ids(seqs[:1]).ctypes.data, 1, np.array(members, np.int64).ctypes.data,
                                    np.array(keys, np.int64).ctypes.data, 1)
        assert y == -1


def test_least_is_a_whole_number_of_any_size():
    cache, seqs, _ = _forks()
    for least, longest in ((0, 640), (256, 640), (688, 640), (689, 0), (1 << 31, 0), (1 << 63, 0), (1 << 64, 0), ((1 << 64) + 5, 0)):
        assert cache.shared(seqs, 8, least=least).longest == longest
    for least in (-1, -(1 << 63) - 1, -(1 << 64)):
        with pytest.raises(ValueError):
            cache.shared(seqs, 8, least=least)
    for least in (2.5, None, "3"):
        with pytest.raises(TypeError):
            cache.shared(seqs, 8, least=least)


def test_the_largest_group():
    """2^27 - 1 sequences of 16 heads: the plan's tiles are counted to the end."""
    from respect_amd import _lib
    _forks()
    most = 2 ** 27 - 1
    for members, tiles in (([most], 2 ** 24), ([most - 1], 2 ** 24), ([5, most - 5], 2 ** 24), ([most - 8], 2 ** 24 - 1),
                           ([most + 1], -1), ([most, 1], -1)):
        m, k = np.array(members, np.int64), np.full(len(members), 100, np.int64)
        want = tiles if len(members) == 1 or tiles < 0 else 1 + 2 ** 24
        assert _lib.lib().rspx_shared_plan(m.ctypes.data, k.ctypes.data, len(m), 16, None, None) == want, members


# ------------------------------------------------------------------ on the GPU

CFG = dict(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=4096)


@pytest.fixture(scope="module")
def model():
    from respect_amd.decoding.engine import Decoder, DecoderConfig
    return Decoder(DecoderConfig(**CFG), seed=1, std=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_steps_refuse_a_plan_that_is_not_theirs(model, fmt):
    """Another order, another document's forks, a first fork that was cut back and has grown again: refused,
    with the books as they were; one that is still short is taken by itself."""
    from respect_amd.decoding.paged_kv import PagedKVCache
    cache = PagedKVCache(CFG["layers"], CFG["kv_heads"], CFG["head_dim"], 400, page=16, dtype=fmt)
    g = torch.Generator().manual_seed(0)
    docs = [torch.randint(0, CFG["vocab"], (n,), generator=g).cuda() for n in (530, 600)]
    (a, b), _ = model.prefill_batch(docs, cache)
    fa, fb = cache.fork([a], 3), cache.fork([b], 3)
    tokens = torch.tensor([1, 2, 3, 4, 5, 6], device="cuda")
    plan = cache.shared(fa + fb, CFG["heads"])
    assert plan.members == [3, 3] and plan.longest == 576

    def refused(seqs):
        free, lengths = cache.free_pages, [cache.length(s) for s in seqs]
        with pytest.raises(ValueError):
            model.step_batch(tokens, cache, seqs, shared=plan)
        assert (cache.free_pages, [cache.length(s) for s in seqs]) == (free, lengths)
    for seqs in ([fa[0], fb[0], fa[1], fb[1], fa[2], fb[2]], [*fa[:2], fb[0], fa[2], *fb[1:]]):
        refused(seqs)
    copy = cache.fork(fa + fb)
    alone = cache.fork(fa[:1])
    cache.compact([fa[0]], 100, [[]])
    cache.compact(alone, 100, [[]])
    rest = cache.shared(copy[1:], CFG["heads"])
    assert rest.members == [2, 3] and rest.longest == 576
    got = model.step_batch(tokens, cache, fa + fb, shared=plan)
    assert torch.equal(got[1:], model.step_batch(tokens[1:], cache, copy[1:], shared=rest))
    assert torch.equal(got[:1], model.step_batch(tokens[:1], cache, alone))
    cache.extend([fa[0]], 410)                                   # 511 rows: the next step has as many as are shared
    refused(fa + fb)
    cache.free([a, b, *fa, *fb, *copy, *alone])
    assert cache.free_pages == 400


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
