"""The native form of the serving operators' common case (respect_amd/_calls): what it leaves to
the Python wrappers, and that both give the same results."""
import pytest
import torch

BF = torch.bfloat16


def test_calls_leaves_what_it_does_not_take():
    from respect_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    c = _lib.calls()
    x, i = torch.zeros(4, 2, 64, dtype=BF), torch.zeros(1, 4, dtype=torch.int32)
    assert c.prompt_attn(x, x, x, 4, 4, i, i, i, None) is None and c.prompt_attn(x) is None
    assert c.paged_attn(x, x, x, i, i[0], 16, None) is None and c.paged_attn() is None
    f = torch.zeros(2, 8)
    assert c.token_logprobs(f, torch.zeros(2, dtype=torch.int64), 1, 0, 0) is None
    assert c.token_logprobs(f, f, 1.5, None, "a") is None


def test_sizes_past_32_bits_are_refused():
    """Tensors of one element seen 2^32 times over: their sizes are refused, not cut to 32 bits."""
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache
    from respect_amd.kernels.paged_attention import paged_attn
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn
    if not _lib.LIB_PATH.exists():
        pytest.skip("librespect_amd.so not built")
    big = 1 << 32
    q, kc, table, lens = (torch.zeros(1, 4, 64, dtype=BF), torch.zeros(2, 64, 64, dtype=BF),
                          torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    for args in ((q.expand(1, -1, -1), kc[:, :1].expand(2, big + 64, 64), table),
                 (q, kc[:1].expand(big + 2, 64, 64), table), (q[:, :1].expand(1, big + 4, 64), kc, table),
                 (q, kc, table[:, :1].expand(1, big + 4))):
        with pytest.raises(ValueError, match="2\\^31"):
            paged_attn(args[0], args[1], args[1], args[2], lens, 16)
    x = torch.zeros(4, 1, 64, dtype=BF)
    for h, hk in ((big + 4, 2), (4, big + 2)):
        with pytest.raises(ValueError, match="2\\^31"):
            prompt_attn(x.expand(4, h, 64), x.expand(4, hk, 64), x.expand(4, hk, 64), PackedPrompts([4], device="cpu"))
    c = PagedKVCache(1, 1, 8, pages=4, page=4, device="cpu")
    row = torch.zeros(1, 1, 8, dtype=BF).expand(big + 1, 1, 8)
    with pytest.raises(ValueError, match="2\\^31"):
        c.write(0, row, row, torch.zeros(1, dtype=torch.int32).expand(big + 1))


@pytest.mark.gpu
def test_calls_equal_the_wrappers_own_path(monkeypatch):
    from respect_amd import _lib
    from respect_amd.decoding.logprobs import token_logprobs
    from respect_amd.kernels.paged_attention import paged_attn
    from respect_amd.kernels.prompt_attention import PackedPrompts, prompt_attn

    class Leave:
        def __getattr__(self, name):
            return lambda *a: None

    g = torch.Generator(device="cuda")
    g.manual_seed(1)

    def r(*s, dtype=BF):
        return torch.randn(*s, generator=g, device="cuda").to(dtype)

    q, k, v, plan = r(70, 8, 64), r(90, 2, 64), r(90, 2, 64), PackedPrompts([60, 10], [60, 30])
    kc = r(2, 640, 64)
    table = torch.randperm(40, generator=g, device="cuda").to(torch.int32).view(2, 20)
    lens = torch.tensor([311, 7], dtype=torch.int32, device="cuda")
    x, t = r(3, 5000, dtype=torch.float32), torch.tensor([1, 2, 3], device="cuda")
    wide = r(4, 70, 8, 64)
    calls = [
        (True, lambda: prompt_attn(q, k, v, plan)),
        (True, lambda: prompt_attn(wide[2], k, v, plan, sm_scale=0.3)),
        (False, lambda: prompt_attn(r(70, 8, 72)[:, :, 3:67], k, v, plan)),
        (True, lambda: paged_attn(q[:2], kc, kc, table, lens, 16)),
        (True, lambda: paged_attn(q[:2], kc, kc, table, lens, 16, sm_scale=1)),
        (False, lambda: paged_attn(q[:2], kc, kc, table.t().contiguous().t(), lens, 16)),
        (True, lambda: token_logprobs(x, t)),
        (True, lambda: token_logprobs(x, t, top=9, offset=3, size=40)),
        (True, lambda: token_logprobs(x[:, 1:], t, top=9)),
        (False, lambda: token_logprobs(x[:1].expand(3, 5000), t, top=9)),
        (False, lambda: token_logprobs(x[0].as_strided((1, 5000), (0, 1)), t[:1], top=9)),
    ]
    native = _lib.calls()
    for taken, call in calls:
        got = []

        class Watch:
            def __getattr__(self, name):
                def f(*a):
                    y = getattr(native, name)(*a)
                    got.append(y is not None)
                    return y
                return f
        state = g.get_state()
        with monkeypatch.context() as m:
            m.setattr(_lib, "_calls", Watch())
            a = call()
        assert got == [taken]
        g.set_state(state)
        with monkeypatch.context() as m:
            m.setattr(_lib, "_calls", Leave())
            b = call()
        for y, z in zip(*(((a,), (b,)) if isinstance(a, torch.Tensor) else (a, b))):
            assert y.shape == z.shape and y.dtype == z.dtype and torch.equal(y, z)


@pytest.mark.gpu
def test_pages_calls_equal_the_wrappers_own_path(monkeypatch):
    """The same run of bookkeeping calls natively and through the wrapper: pools, tables, slots and
    errors are the same; tuples, ranges and numpy numbers are left to the wrapper."""
    import numpy as np
    from respect_amd import _lib
    from respect_amd.decoding.paged_kv import PagedKVCache

    class Leave:
        def __getattr__(self, name):
            return lambda *a: None

    def play():
        c = PagedKVCache(2, 2, 64, pages=30, page=4, sequences=9)
        g = torch.Generator(device="cuda")
        g.manual_seed(0)
        for t in c.k + c.v:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        out = []
        seqs = c.add([9, 4, 13])
        out.append(c.fork(seqs, 2))
        c.extend(out[0][:2], [3, 1])
        c.extend(range(3))
        c.compact(seqs, [1, 0, 6], [[0, 2, 5], [], [3, 4]])
        c.compact(np.array(out[0][:1]), 2, [range(1, 4)])
        out += [c.slots(seqs, 0, [2, 0, 3]).tolist(), c.slots(tuple(seqs), [1, 0, 1], 0).tolist()]
        table, lens = c.tables(seqs + out[0])
        out += [table.tolist(), lens.tolist(), c.free_pages]
        for call in (lambda: c.fork([77]), lambda: c.fork(seqs, 9), lambda: c.extend(seqs, -1), lambda: c.extend(seqs, 500),
                     lambda: c.compact(seqs, 0, [[0]]), lambda: c.compact(seqs, 0, [[9], [], []]), lambda: c.tables([-1]),
                     lambda: c.slots(seqs, 0, 99), lambda: c.slots([seqs[0]], -1, 1), lambda: c.fork([1 << 70])):
            with pytest.raises((ValueError, RuntimeError, OverflowError)) as e:
                call()
            out.append(type(e.value))
        for bad in ([77], [seqs[0], seqs[0]], [1 << 70]):
            with pytest.raises((ValueError, RuntimeError, OverflowError)) as e:
                c.free(bad)
            out.append(type(e.value))
        c.free(out[0][2:4])
        c.free(tuple(seqs[:1]))
        c.free([])
        out += [c.free_pages, c.add([1, 1, 1])]
        return out, [t.clone() for t in c.k + c.v]
    a, ta = play()
    with monkeypatch.context() as m:
        m.setattr(_lib, "_calls", Leave())
        b, tb = play()
    assert a == b and all(torch.equal(x, y) for x, y in zip(ta, tb))
