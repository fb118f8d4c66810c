"""Attention over packed whole prompts (kernels.prompt_attention) against 64-bit attention
per sequence: grouped heads, lengths from nothing to some hundred, earlier keys, rows that
see nothing, strided inputs, values that are not finite behind a row; a row's bits do not
depend on the pack; refusals on the CPU."""
import numpy as np
import pytest
import torch

BF = torch.bfloat16


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _inputs(rows, keys, H, HK, D, seed=0):
    g = _gen(seed)
    q = torch.randn(sum(rows), H, D, generator=g).to(BF)
    k, v = (torch.randn(sum(keys), HK, D, generator=g).to(BF) for _ in range(2))
    return q, k, v


def _exact(q, k, v, rows, keys, scale=None):
    """(result, bound) in float64.  The bound, to first order: every p rounded to bf16 (half a
    step, d_i <= 2^-8 of it) in numerator and denominator alike, so that the result moves by
    sum p_i d_i v_i - o sum p_i d_i = sum p_i d_i (v_i - o), and the result once; scores accumulated over D products and sums over n
    keys in fp32, whose steps are 2^-24 each; a score's error moves p by that much relative,
    in the numerator and in the denominator."""
    T, H, D = q.shape
    G = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, bound = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    t = j = 0
    for n, m in zip(rows, keys):
        for h in range(H):
            qd, kd, vd = q[t:t + n, h].double(), k[j:j + m, h // G].double(), v[j:j + m, h // G].double()
            for i in range(n):
                seen = m - n + i + 1
                if seen <= 0:
                    continue
                s = kd[:seen] @ qd[i] * scale
                p = torch.softmax(s, 0)
                o, a = p @ vd[:seen], p @ vd[:seen].abs()
                es = 2.0 ** -24 * ((D + 8) * float((kd[:seen].abs() @ qd[i].abs()).max()) * scale + 8)
                out[t + i, h] = o
                off = p @ (vd[:seen] - o).abs()
                bound[t + i, h] = (off * 2.0 ** -8 + a * (2 * es + 2 * (seen + 64) * 2.0 ** -24) + o.abs() * 2.0 ** -8) * 1.02
        t, j = t + n, j + m
    return out, bound


def _check(got, want, bound):
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all()
    worst = float((err / (bound + 1e-30)).max()) if err.numel() else 0.0
    print(f"max err / bound {worst:.3f}", flush=True)
    assert worst <= 1


def test_plan_tiles_cover_every_row_once():
    from respect_amd import _lib
    from respect_amd.kernels.prompt_attention import TILE_ROWS, PackedPrompts
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    rows, keys = [0, 5, 64, 1, 131, 300], [7, 5, 10, 1, 200, 300]
    plan = PackedPrompts(rows, keys, device="cpu")
    assert (plan.Tq, plan.Tk, plan.rows, plan.keys) == (sum(rows), sum(keys), rows, keys)
    for size, tiles in zip(TILE_ROWS, plan._lists):
        t = tiles.numpy().astype(np.int64)
        sees = np.full(plan.Tq, -10 ** 9)
        first = np.full(plan.Tq, -1)
        for q0, n, k0, seen in t:
            assert 0 < n <= size
            assert (first[q0:q0 + n] == -1).all()
            first[q0:q0 + n] = k0
            sees[q0:q0 + n] = seen + np.arange(n)
        q0 = k0 = 0
        for n, m in zip(rows, keys):
            assert (first[q0:q0 + n] == k0).all() and (sees[q0:q0 + n] == m - n + 1 + np.arange(n)).all()
            q0, k0 = q0 + n, k0 + m
        assert (np.diff(t[:, 1] + t[:, 3]) <= 0).all()
    got = [_lib.lib().rspx_prompt_attn_tile_rows(h, hk) for h, hk in ((32, 8), (16, 2), (4, 2), (6, 2), (5, 5))]
    assert got == [32, 32, 64, 128, 128]
    assert PackedPrompts([], device="cpu").Tq == 0 and len(PackedPrompts([0, 0], device="cpu")._lists[0]) == 0


def test_refusals():
    from respect_amd import _lib
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    for bad in (([1, -1], None), ([1, 2], [1]), ([1 << 31], None), ([1 << 30] * 2, [0, 0]), ([1, 1], [1 << 30, 1 << 30])):
        with pytest.raises(ValueError):
            PackedPrompts(*bad, device="cpu")
    plan = PackedPrompts([4], device="cpu")
    q, k, v = _inputs([4], [4], 4, 2, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        prompt_attn(q, k, v, plan)
    with pytest.raises(ValueError):
        prompt_attn(q, k, v[:, :1], plan)
    with pytest.raises(ValueError):
        prompt_attn(q[:3], k, v, plan)
    with pytest.raises(ValueError):
        prompt_attn(q[:, :3], k, v, plan)
    L = _lib.lib()

    def call(H=4, HK=2, Tq=4, Tk=4, D=64, scale=0.1, p=16, st=256, n=1, skt=256):
        return L.rspx_prompt_attn(p, st, 64, p, skt, 64, p, 256, 64, 16, n, p, st, 64, H, HK, Tq, Tk, D, scale, None)
    assert call(H=3) == -1 and call(Tq=-1) == -1 and call(scale=0.0) == -1 and call(scale=-1.0) == -1
    assert call(scale=float("nan")) == -1 and call(scale=float("inf")) == -1
    assert call(skt=1 << 24) == -1 and call(p=0) == -1
    assert call(D=96) == -2
    assert call(p=8) == -4 and call(st=100) == -4
    assert call(n=0) == 0 and call(Tq=0) == 0
    assert L.rspx_prompt_attn_tile_rows(3, 2) == -1 and L.rspx_prompt_attn_tile_rows(0, 1) == -1


def test_lengths_that_are_not_whole_are_refused():
    from respect_amd import _lib
    from respect_amd.kernels.prompt_attention import PackedPrompts
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    for bad in (([1.9], None), ([2, 1.0], None), ([2], [2.5]), (np.array([1.5]), None), (["3"], None), ([[1, 2]], None)):
        with pytest.raises(TypeError):
            PackedPrompts(*bad, device="cpu")
    plan = PackedPrompts(np.array([3, 1], np.int16), torch.tensor([5, 1]), device="cpu")
    assert plan.rows == [3, 1] and plan.keys == [5, 1]


SHAPES = [(8, 2, 128), (4, 2, 64), (3, 1, 128), (16, 2, 64), (4, 1, 32), (4, 1, 256), (2, 2, 256), (6, 2, 64)]
PACKS = [([1], None), ([77], None), ([64, 65, 1, 0, 130], None), ([33, 5], [97, 5]), ([40, 7, 3], [10, 7, 0]),
         ([129], [323])]


@pytest.mark.gpu
@pytest.mark.parametrize("H,HK,D", SHAPES)
@pytest.mark.parametrize("pack", range(len(PACKS)))
def test_against_64_bits(H, HK, D, pack):
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    rows, keys = PACKS[pack]
    keys = rows if keys is None else keys
    q, k, v = _inputs(rows, keys, H, HK, D, seed=pack)
    plan = PackedPrompts(rows, keys)
    got = prompt_attn(q.cuda(), k.cuda(), v.cuda(), plan)
    assert got.shape == q.shape and got.dtype == BF
    _check(got, *_exact(q, k, v, rows, keys))
    t = 0
    for n, m in zip(rows, keys):   # rows that see no key
        assert (got[t:t + max(0, min(n, n - m))] == 0).all()
        t += n


@pytest.mark.gpu
def test_scale_large_scores_and_out():
    """A scale of the caller's, scores of some hundred (the running maximum moves often), a result
    written in place between rows that keep what they held."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    rows = [100, 201]
    q, k, v = _inputs(rows, rows, 4, 1, 64, seed=3)
    k = (k.float() * torch.linspace(0.1, 12, sum(rows))[:, None, None]).to(BF)
    out = torch.full((sum(rows) + 2, 4, 64), 7.0, dtype=BF, device="cuda")
    got = prompt_attn(q.cuda(), k.cuda(), v.cuda(), PackedPrompts(rows), sm_scale=1.5, out=out[1:-1])
    assert got.data_ptr() == out[1:].data_ptr() and (out[0] == 7).all() and (out[-1] == 7).all()
    _check(got, *_exact(q, k, v, rows, rows, 1.5))


@pytest.mark.gpu
@pytest.mark.parametrize("H,HK,D", [(8, 2, 128), (4, 2, 64), (3, 3, 128)])
def test_rows_do_not_depend_on_the_pack(H, HK, D):
    """A sequence alone, packed between others, cut short, in views with other strides, and with
    what lies behind a row replaced: the same bits."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    rows = [50, 200, 3, 170]
    q, k, v = (t.cuda() for t in _inputs(rows, rows, H, HK, D, seed=5))
    all_ = prompt_attn(q, k, v, PackedPrompts(rows))
    a, b = 50, 250
    alone = prompt_attn(q[a:b].clone(), k[a:b].clone(), v[a:b].clone(), PackedPrompts([200]))
    assert torch.equal(alone, all_[a:b])
    short = prompt_attn(q[a:a + 71], k[a:a + 71], v[a:a + 71], PackedPrompts([71]))
    assert torch.equal(short, all_[a:a + 71])
    last = prompt_attn(q[b - 9:b], k[a:b], v[a:b], PackedPrompts([9], [200]))
    assert torch.equal(last, all_[b - 9:b])
    # One packed projection [T, (H + 2 HK) D], head-major keys, values in a wider row.
    qkv = torch.cat((q.flatten(1), k.flatten(1), v.flatten(1)), 1)
    qs = qkv[:, :H * D].view(-1, H, D)
    ks = k.transpose(0, 1).contiguous().transpose(0, 1)
    vs = qkv[:, (H + HK) * D:].view(-1, HK, D)
    assert qs.data_ptr() == qkv.data_ptr()
    assert torch.equal(prompt_attn(qs, ks, vs, PackedPrompts(rows)), all_)


@pytest.mark.gpu
@pytest.mark.parametrize("H,HK,D", [(4, 1, 128), (4, 2, 64), (2, 2, 32), (8, 2, 256)])
def test_chunks_give_the_bits_of_the_whole_prompt(H, HK, D):
    """A prompt in one pass, and in chunks after its earlier keys, between other sequences: a row
    falls in other tiles, and steps that a tile sees whole are seen in part elsewhere.  Scores
    that grow and fall, so that the running maximum moves in every kind of step."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    n = 700
    q, k, v = _inputs([n], [n], H, HK, D, seed=21)
    k = (k.float() * (1 + 5 * torch.sin(torch.arange(n) / 37.0).abs())[:, None, None]).to(BF)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    whole = prompt_attn(q, k, v, PackedPrompts([n]))
    for chunk in (1, 64, 100, 333):
        ends = list(range(chunk, n, chunk)) + [n] if chunk > 1 else [1, 64, 65, 128, 129, 640, 700]
        firsts = [max(0, e - chunk) for e in ends] if chunk == 1 else [0] + ends[:-1]
        rows = [e - f for f, e in zip(firsts, ends)]
        qs = torch.cat([q[f:e] for f, e in zip(firsts, ends)])
        ks, vs = (torch.cat([t[:e] for e in ends]) for t in (k, v))
        got = prompt_attn(qs, ks, vs, PackedPrompts(rows, ends))
        want = torch.cat([whole[f:e] for f, e in zip(firsts, ends)])
        assert torch.equal(got, want), chunk


@pytest.mark.gpu
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_values_behind_a_row_do_not_reach_it(what, D):
    """K and V of one token that are not finite: every earlier row keeps its bits, every row of
    the other sequences too, and the later ones are not finite in those columns."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    rows = [90, 150, 40]
    q, k, v = (t.cuda() for t in _inputs(rows, rows, 4, 1, D, seed=8))
    plan = PackedPrompts(rows)
    ref = prompt_attn(q, k, v, plan)
    for at in (0, 31, 64, 100, 127, 149):
        v2 = v.clone()
        v2[90 + at, 0, 5] = what
        got = prompt_attn(q, k, v2, plan)
        assert torch.equal(got[:90 + at], ref[:90 + at]) and torch.equal(got[240:], ref[240:])
        assert not torch.isfinite(got[90 + at:240, :, 5]).any()
        assert torch.isfinite(got[90 + at:240, :, 6:]).all() and torch.isfinite(got[90 + at:240, :, :5]).all()
        k2 = k.clone()
        k2[90 + at, 0] = what
        got = prompt_attn(q, k2, v, plan)
        assert torch.equal(got[:90 + at], ref[:90 + at]) and torch.equal(got[240:], ref[240:])


@pytest.mark.gpu
def test_long_many_heads_spot_rows():
    """A long prompt beside short ones at the 8B heads: rows at its ends and middle, against 64 bits."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    rows, H, HK, D = [3, 2500, 61], 32, 8, 128
    q, k, v = _inputs(rows, rows, H, HK, D, seed=9)
    got = prompt_attn(q.cuda(), k.cuda(), v.cuda(), PackedPrompts(rows)).cpu()
    for i in (0, 1, 63, 64, 1250, 2047, 2048, 2499):
        a, b = 3, 3 + i + 1
        want, bound = _exact(q[b - 1:b], k[a:b], v[a:b], [1], [i + 1])
        _check(got[b - 1:b], want, bound)


@pytest.mark.gpu
def test_graph_replays_and_streams():
    """Captured and replayed on changed inputs, between eager calls on another stream."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    rows = [70, 33]
    plan = PackedPrompts(rows)
    q, k, v = (t.cuda() for t in _inputs(rows, rows, 8, 2, 128))
    prompt_attn(q, k, v, plan)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = prompt_attn(q, k, v, plan)
        with pytest.raises(RuntimeError, match="captured"):
            PackedPrompts(rows)
    side = torch.cuda.Stream()
    for seed in range(3):
        for t, x in zip((q, k, v), _inputs(rows, rows, 8, 2, 128, seed=20 + seed)):
            t.copy_(x)
        g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = prompt_attn(q, k, v, plan)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, eager)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_gpu_refusals_and_empty():
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    q, k, v = (t.cuda() for t in _inputs([4], [4], 4, 2, 64))
    with pytest.raises(TypeError):
        prompt_attn(q.float(), k, v, PackedPrompts([4]))
    with pytest.raises(RuntimeError):
        prompt_attn(q, k, v, PackedPrompts([4], device="cpu"))
    with pytest.raises(RuntimeError):
        prompt_attn(q[..., :24].contiguous(), k[..., :24].contiguous(), v[..., :24].contiguous(), PackedPrompts([4]))
    with pytest.raises(TypeError):
        prompt_attn(q, k, v, PackedPrompts([4]), out=torch.empty(4, 4, 64, device="cuda"))
    with pytest.raises(ValueError):
        prompt_attn(q, k, v, PackedPrompts([4]), out=torch.empty(5, 4, 64, dtype=BF, device="cuda"))
    with pytest.raises(RuntimeError):
        prompt_attn(q, k, v, PackedPrompts([4]), sm_scale=0.0)
    assert prompt_attn(q[:0], k[:0], v[:0], PackedPrompts([])).shape == (0, 4, 64)
    assert (prompt_attn(q, k[:0], v[:0], PackedPrompts([4], [0])) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("H,HK,D", [(4, 1, 128), (4, 2, 64), (2, 2, 32), (8, 2, 256)])
def test_values_that_are_not_finite_in_whole_and_partial_steps(what, H, HK, D):
    """Two values that are not finite, one behind a score so low that p is 0 in fp32 (0 times it is
    NaN), one with an ordinary p: a row has the same result whether its tile sees their steps whole
    (the prompt in one pass) or in part or last (the row alone after its earlier keys)."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    n = 200
    q, k, v = _inputs([n], [n], H, HK, D, seed=31)
    q = q.abs()
    k[5] = -200.0
    v[5, :, 3], v[70, :, 4] = what, what
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    whole = prompt_attn(q, k, v, PackedPrompts([n])).float()
    assert torch.isfinite(whole[:5]).all() and torch.isfinite(whole[:70, :, 4]).all()
    assert torch.isnan(whole[6:, :, 3]).all()
    want = torch.full_like(whole[70:, :, 4], what)
    assert torch.equal(whole[70:, :, 4].nan_to_num(7.0), want.nan_to_num(7.0))
    rest = [d for d in range(D) if d not in (3, 4)]
    assert torch.isfinite(whole[:, :, rest]).all()
    for end in (5, 6, 7, 40, 64, 65, 71, 128, 129, 192, 200):
        one = prompt_attn(q[end - 1:end], k[:end], v[:end], PackedPrompts([1], [end])).float()[0]
        assert torch.equal(torch.isnan(one), torch.isnan(whole[end - 1])), end
        assert torch.equal(one.nan_to_num(7.0), whole[end - 1].nan_to_num(7.0)), end


@pytest.mark.gpu
@pytest.mark.parametrize("H,HK,D", [(8, 2, 128), (2, 2, 64), (4, 2, 256)])
def test_result_in_place_of_q(H, HK, D):
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    rows = [300, 1, 77]
    q, k, v = (t.cuda() for t in _inputs(rows, rows, H, HK, D, seed=17))
    plan = PackedPrompts(rows)
    want = prompt_attn(q, k, v, plan)
    assert prompt_attn(q, k, v, plan, out=q) is q and torch.equal(q, want)


@pytest.mark.gpu
def test_more_workgroups_than_a_grid_holds():
    """32900 one-token sequences of 512 heads: 16.8 M workgroups, more than the 2^32 threads of a grid
    dimension, whose count would start again at 0; every result is its one value."""
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    n = 32900
    x = torch.randn(n, 512, 32, device="cuda").to(BF)
    assert torch.equal(prompt_attn(x, x, x, PackedPrompts([1] * n)), x)


def test_more_heads_than_a_grid_holds_are_refused():
    from respect_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    for H, want in ((1 << 23, 0), ((1 << 23) + 1, -2), ((1 << 31) - 1, -2)):
        got = _lib.lib().rspx_prompt_attn(16, 64, 64, 16, 64, 64, 16, 64, 64, 16, 0 if want == 0 else 1, 16, 64, 64, H, H, 4, 4,
                                          64, 0.1, None)
        assert got == want
