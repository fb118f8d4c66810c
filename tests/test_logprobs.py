"""Log probabilities of given tokens, entropy and best alternatives (decoding.logprobs)
against 64 bits: vocabularies that end inside a chunk, ties, excluded columns, infinities and
NaN, rows with nothing left, tokens that are none, strided rows; refusals on the CPU."""
import math

import pytest
import torch


def _logits(M, V, seed=0, scale=2.5):
    g = torch.Generator()
    g.manual_seed(seed)
    x = torch.randn(M, V, generator=g) * scale
    t = torch.randint(0, V, (M,), generator=g)
    x[torch.arange(M), t] += 6
    return x, t


def _exact(x, t, top, off=0, size=0):
    """Results in float64 and bounds.  With d_j = x_j - m: d is rounded once, so is d log2 e, whose
    constant is off by 0.22 of 2^-24; each moves e^d by |d| 2^-24 relative, and 2^x itself is off by
    a unit: (2.25 |d| + 8) 2^-24 for an element of z.  Its sums over 16 elements and the 6 steps
    of a wave add 22 * 2^-24; the waves' steps are joined in 64 bits and every result is rounded once.
    u = sum e d carries the same error on each term, one more d and one more product."""
    x = x.double().clone()
    x[:, off:off + size] = -math.inf
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    m = x.max(-1, keepdim=True).values
    d = torch.where(p > 0, m - x, torch.zeros_like(x))
    eps = 2.0 ** -24
    ez = eps * (40 + 2.25 * (p * d).sum(-1))
    given = lp.gather(1, t[:, None])[:, 0]
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    eh = ez + eps * ((p * d * (42 + 2.25 * d)).sum(-1) + (p * d).sum(-1) * (40 + 2.25 * (p * d).sum(-1)))
    ids = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :top]
    values = lp.gather(1, ids)
    return (given, ez + eps * given.abs()), (entropy, eh + eps * entropy.abs()), (values, ez[:, None] + eps * values.abs()), ids


def _check(got, want):
    for name, a, (b, bound) in zip(("given", "entropy", "values"), got[:3], want[:3]):
        a = a.double().cpu()
        same = torch.isinf(b) | torch.isnan(b)
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        assert torch.equal(a[same & ~torch.isnan(b)], b[same & ~torch.isnan(b)]), name
        err = ((a - b).abs() / (bound + 1e-30))[~same]
        print(name, float(err.max()) if err.numel() else 0.0, flush=True)
        assert (err <= 1).all(), name
    assert torch.equal(got[3].cpu(), want[3])


def test_refusals():
    from respect_amd import _lib
    from respect_amd.decoding.logprobs import token_logprobs
    x, t = _logits(2, 100)
    with pytest.raises(TypeError):
        token_logprobs(x, t)                 # not on a GPU
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    L = _lib.lib()

    def call(M=2, V=100, sl=100, off=0, size=0, top=5, p=16, ws=1 << 20, wp=16, t=16):
        return L.rspx_token_logprobs(p, sl, M, V, off, size, t, top, 16, 16, 16, 16, wp, ws, None)
    assert call(M=-1) == -1 and call(V=0) == -1 and call(sl=96) == -1 and call(off=-1) == -1 and call(size=-1) == -1
    assert call(top=-1) == -1 and call(V=3, top=4) == -1 and call(p=0) == -1 and call(t=0) == -1
    assert call(top=65) == -2 and call(V=(1 << 30) + 4, sl=(1 << 30) + 4) == -2
    assert call(p=18) == -4 and call(wp=20) == -4
    assert call(ws=64) == -3 and call(wp=0) == -3
    assert call(M=0) == 0
    assert L.rspx_token_logprobs_workspace_bytes(1, 0, 1) == -1
    assert L.rspx_token_logprobs_workspace_bytes(1, 5, 65) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 4095, 4096, 4097, 8193, 50257, 151936])
@pytest.mark.parametrize("top", [0, 1, 5, 64])
def test_against_64_bits(V, top):
    from respect_amd.decoding.logprobs import token_logprobs
    x, t = _logits(3, V, seed=V)
    got = token_logprobs(x.cuda(), t.cuda(), top=top)
    n = min(top, V)
    assert got[0].shape == got[1].shape == (3,) and got[2].shape == got[3].shape == (3, n) and got[3].dtype == torch.int64
    _check(got, _exact(x, t, n))


@pytest.mark.gpu
@pytest.mark.parametrize("top", [1, 20, 64])
def test_ties_and_sorted_rows(top):
    """All equal, few distinct values, -0 and +0, sorted up and down, one thread's elements the best."""
    from respect_amd.decoding.logprobs import token_logprobs
    V = 10000
    g = torch.Generator()
    g.manual_seed(1)
    x = torch.stack([torch.zeros(V), torch.randint(0, 3, (V,), generator=g).float(), -torch.arange(V) / 100.0,
                     torch.arange(V) / 100.0, torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0),
                     torch.where(torch.arange(V) % 1024 < 4, 5.0 + torch.arange(V) / V, 0.0)])
    t = torch.tensor([0, V - 1, 5, 7, 9, 4096])
    _check(token_logprobs(x.cuda(), t.cuda(), top=top), _exact(x, t, top))


@pytest.mark.gpu
def test_excluded_columns_masks_and_lowest_values():
    from respect_amd.decoding.logprobs import token_logprobs
    x, t = _logits(6, 9001, seed=3)
    x[0, 100:] = -math.inf                      # whole chunks masked
    x[1, :8200] = -math.inf
    x[2] = torch.finfo(torch.float32).min       # all of the type's lowest value: all equal
    x[3, 1:] = torch.finfo(torch.float32).min   # one score left
    t[0], t[1], t[4] = 8000, 8999, 10           # the first two: masked, open
    _check(token_logprobs(x.cuda(), t.cuda(), top=30), _exact(x, t, 30))
    t[5] = 4100
    _check(token_logprobs(x.cuda(), t.cuda(), top=30, offset=4090, size=1000), _exact(x, t, 30, 4090, 1000))
    _check(token_logprobs(x.cuda(), t.cuda(), top=3, offset=8990, size=10 ** 6), _exact(x, t, 3, 8990, 10 ** 6))


@pytest.mark.gpu
def test_rows_that_are_not_finite():
    """NaN and +inf rows, rows with nothing left, tokens outside the vocabulary."""
    from respect_amd.decoding.logprobs import token_logprobs
    V = 5000
    x, t = _logits(7, V, seed=4)
    x[0, 4500] = math.nan
    x[1, 3] = math.inf
    x[2] = -math.inf
    x[5] = math.nan
    x[6, :4096] = -math.inf
    x[6, 4200] = math.nan
    t[3], t[4] = -1, V
    given, entropy, values, ids = (a.cpu() for a in token_logprobs(x.cuda(), t.cuda(), top=4))
    bad = [0, 1, 5, 6]
    assert torch.isnan(given[bad]).all() and torch.isnan(entropy[bad]).all() and torch.isnan(values[bad]).all()
    assert ids[0, 0] == 4500 and ids[1, 0] == 3 and ids[5].tolist() == [0, 1, 2, 3] and ids[6, 0] == 4200
    assert ids[0, 1:].tolist() == torch.argsort(x[0].nan_to_num(-100.0), descending=True)[:3].tolist()
    assert given[2] == -math.inf and entropy[2] == 0 and (values[2] == -math.inf).all() and ids[2].tolist() == [0, 1, 2, 3]
    assert torch.isnan(given[3:5]).all() and torch.isfinite(entropy[3:5]).all() and torch.isfinite(values[3:5]).all()
    # everything excluded
    given, entropy, values, ids = token_logprobs(x[3:5].cuda(), t[:2].cuda(), top=2, size=V)
    assert (given == -math.inf).all() and (entropy == 0).all() and (values == -math.inf).all()


@pytest.mark.gpu
def test_rows_do_not_depend_on_the_batch_and_agree_with_greedy():
    """A row's bits alone, in a batch, in a padded and in a misaligned view; its best column is the
    greedy token; two calls at once on two streams and a replayed graph give the same."""
    from respect_amd.decoding.acceptance import greedy_token
    from respect_amd.decoding.logprobs import token_logprobs
    x, t = (a.cuda() for a in _logits(5, 20004, seed=6))
    ref = token_logprobs(x, t, top=7, offset=50, size=60)
    assert torch.equal(ref[3][:, 0], greedy_token(x, 50, 60))
    one = token_logprobs(x[2:3], t[2:3], top=7, offset=50, size=60)
    assert all(torch.equal(a[0], b[2]) for a, b in zip(one, ref))
    pad = torch.full((5, 20100), math.nan, device="cuda")
    for shift in (0, 1, 4):
        pad[:, shift:shift + 20004] = x
        got = token_logprobs(pad[:, shift:shift + 20004], t, top=7, offset=50, size=60)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token_logprobs(x, t, top=7, offset=50, size=60)
    side = torch.cuda.Stream()
    for seed in range(3):
        x.copy_(_logits(5, 20004, seed=30 + seed)[0])
        side.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(side):
            other = token_logprobs(x, t, top=7, offset=50, size=60)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(out, other))
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["spread", "early", "late", "rising", "equal"])
def test_more_alternatives_than_the_join_holds_at_once(where):
    """74 parts of 64 pairs a row, more than the 4096 that the join takes at once: the best of them
    in the parts it takes first, in those it takes last, in both."""
    from respect_amd.decoding.logprobs import token_logprobs
    V, top = 300001, 64
    x, t = _logits(2, V, seed=12)
    if where == "rising":
        x = torch.arange(2 * V).view(2, V) * 2e-4
    elif where == "equal":
        x = torch.zeros(2, V)
    elif where != "spread":
        at = slice(0, 100) if where == "early" else slice(V - 100, V)
        x[:, at] = 20 + torch.arange(100) % 7
    _check(token_logprobs(x.cuda(), t.cuda(), top=top), _exact(x, t, top))


@pytest.mark.gpu
@pytest.mark.parametrize("V,top", [(17, 0), (17, 3), (4100, 2)])
def test_more_rows_than_a_launch_takes(V, top):
    """65540 rows, launched 65535 at a time: rows on both sides of the border against 64 bits, the
    last ones the bits of a call for them alone."""
    from respect_amd.decoding.logprobs import token_logprobs
    M = 65540
    g = torch.Generator(device="cuda")
    g.manual_seed(13)
    x = torch.randn(M, V, generator=g, device="cuda") * 2
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    got = token_logprobs(x, t, top=top, offset=2, size=3)
    some = torch.tensor([0, 1, 40000, 65533, 65534, 65535, 65536, 65539], device="cuda")
    _check([a[some] for a in got], _exact(x[some].cpu(), t[some].cpu(), top, 2, 3))
    alone = token_logprobs(x[65000:], t[65000:], top=top, offset=2, size=3)
    assert all(torch.equal(a, b[65000:]) for a, b in zip(alone, got))


@pytest.mark.gpu
def test_excluded_ranges_past_32_bits():
    """Offsets and sizes that 32 bits do not hold mean what they say; fractions are refused."""
    from respect_amd.decoding.logprobs import token_logprobs
    x, t = _logits(3, 500, seed=11)
    t[0] = 100
    g = (x.cuda(), t.cuda())
    for off, size in ((40, (1 << 32) + 5), (40, 1 << 62), (1 << 32, 60), ((1 << 33) + 7, 1 << 32), (499, 1 << 31)):
        _check(token_logprobs(*g, top=9, offset=off, size=size), _exact(x, t, 9, min(off, 500), size))
    all_ = token_logprobs(*g, top=2, size=1 << 32)
    assert (all_[0] == -math.inf).all() and (all_[1] == 0).all()
    for off, size in ((-(1 << 32), 5), (0, -(1 << 32)), (-1, 1 << 40)):
        with pytest.raises(RuntimeError):
            token_logprobs(*g, offset=off, size=size)
    for off, size in ((1.9, 5), (1, 5.0)):
        with pytest.raises(TypeError):
            token_logprobs(*g, offset=off, size=size)


@pytest.mark.gpu
def test_sizes_past_32_bits_are_refused():
    from respect_amd.decoding.logprobs import token_logprobs
    x, t = torch.zeros(1, 1, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        token_logprobs(x.expand((1 << 32) + 1, 1), t.expand((1 << 32) + 1))
    wide = torch.empty(1, (1 << 32) + 5, device="cuda")   # 17 GB
    with pytest.raises(ValueError):
        token_logprobs(wide, t)
    with pytest.raises((ValueError, RuntimeError)):
        token_logprobs(wide[:, :(1 << 30) + 1], t)


@pytest.mark.gpu
def test_gpu_refusals_and_empty():
    from respect_amd.decoding.logprobs import token_logprobs
    x, t = (a.cuda() for a in _logits(2, 100))
    for args in ((x.half(), t), (x, t.int()), (x, t[:1]), (x, t.cpu()), (x[0], t), (x.t(), t)):
        with pytest.raises(TypeError):
            token_logprobs(*args)
    for top in (-1, 65):
        with pytest.raises(ValueError):
            token_logprobs(x, t, top=top)
    with pytest.raises(RuntimeError):
        token_logprobs(x, t, offset=-1)
    got = token_logprobs(x[:0], t[:0], top=3)
    assert got[0].shape == (0,) and got[2].shape == (0, 3)
