"""The decoder over caches of 8 and 4 bits and over beginnings that sequences share: against the same
decoder over bf16 rows of the same values, against prompts in one piece, a sequence's bits in
different company, and a run of all calls together."""
import pytest
import torch

from _mx import quantise, values

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=4096)
FORMATS = ["bf16", "mxfp8", "mxfp4"]


@pytest.fixture(scope="module")
def model():
    from respect_amd.decoding.engine import Decoder, DecoderConfig
    return Decoder(DecoderConfig(**CFG), seed=1, std=0.05)


def _cache(pages=100, page=16, **kw):
    from respect_amd.decoding.paged_kv import PagedKVCache
    return PagedKVCache(CFG["layers"], CFG["kv_heads"], CFG["head_dim"], pages, page=page, **kw)


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, CFG["vocab"], (n,), generator=g).cuda() for n in lens]


def _tok(*t):
    return torch.tensor(t, device="cuda")


def _close(a, b):
    """Within what separates any two orders of the decoder's sums (test_serving_gpu)."""
    assert torch.isfinite(a).all()
    assert ((a - b).abs().amax(-1) <= 0.05 * b.abs().amax(-1)).all()


def _rounded_cache(fmt):
    """A bf16 cache that keeps the values which ``fmt`` would."""
    from respect_amd.decoding.paged_kv import PagedKVCache

    class Rounded(PagedKVCache):
        def write(self, layer, k, v, slots):
            for x, pool in ((k, self.k[layer]), (v, self.v[layer])):
                pool[:, slots.long()] = values(*quantise(x.cpu(), fmt), fmt).to(torch.bfloat16).cuda().transpose(0, 1)
    cache = Rounded(CFG["layers"], CFG["kv_heads"], CFG["head_dim"], 100, page=16)
    cache.dtype = fmt
    return cache


@pytest.mark.parametrize("fmt", FORMATS[1:])
def test_the_cache_holds_what_the_format_holds(model, fmt):
    """Prefill, further tokens and steps: logits and rows as with a bf16 cache of rounded values."""
    a, b, lens = _cache(dtype=fmt), _rounded_cache(fmt), [100, 1, 37]
    sa, la = model.prefill_batch(_prompts(lens), a)
    sb, lb = model.prefill_batch(_prompts(lens), b)
    assert torch.equal(la, lb)
    for i in range(CFG["layers"]):
        for x, y in zip(a.read(i, a.slots(sa, 0, lens)), b.read(i, b.slots(sb, 0, lens))):
            assert torch.equal(x, y)
    _close(model.append_batch(_prompts([5, 40], 3), a, sa[:2]), model.append_batch(_prompts([5, 40], 3), b, sb[:2]))
    for t in range(3):
        _close(model.step_batch(_tok(t, 7, 9), a, sa), model.step_batch(_tok(t, 7, 9), b, sb))
    assert [a.length(s) for s in sa] == [108, 44, 40]
    f = a.fork(sa[:1], 2)                                        # a begun page moved, codes and scales
    logits = model.step_batch(_tok(5, 5, 5), a, [sa[0], *f])
    assert torch.equal(logits[0], logits[1]) and torch.equal(logits[0], logits[2])
    a.compact([f[0]], 100, [[2, 5]])
    want = a.read(1, a.slots([sa[0]], 102, 1)), a.read(1, a.slots([sa[0]], 105, 1))
    got = a.read(1, a.slots([f[0]], 100, 2))
    for i in range(2):
        assert torch.equal(got[i], torch.cat([want[0][i], want[1][i]]))
    a.free(sa + f)
    assert a.free_pages == 100


@pytest.mark.parametrize("fmt", FORMATS)
def test_further_tokens(model, fmt):
    """Prompts in two pieces: with a bf16 cache the logits of one piece; the bits do not depend on the
    batch, on the pages, or on the sequences that share the first piece."""
    lens, more = [100, 1, 37, 260], [3, 64, 1, 20]
    p, m = _prompts(lens), _prompts(more, 5)
    cache = _cache(dtype=fmt)
    seqs, _ = model.prefill_batch(p, cache)
    got = model.append_batch((x for x in m), cache, seqs)        # prompts from a generator
    assert [cache.length(s) for s in seqs] == [a + b for a, b in zip(lens, more)]
    if fmt == "bf16":
        whole = _cache()
        ws, want = model.prefill_batch([torch.cat(x) for x in zip(p, m)], whole)
        _close(got, want)
        _close(model.step_batch(_tok(1, 2, 3, 4), cache, seqs), model.step_batch(_tok(1, 2, 3, 4), whole, ws))
    for i in (0, 1, 3):
        other = _cache(page=64, pages=20, dtype=fmt)
        (s,), _ = model.prefill_batch(p[i:i + 1], other)
        f = other.fork([s], 2)
        one = model.append_batch([m[i], m[2], m[i]], other, [f[1], s, f[0]])
        assert torch.equal(one[0], got[i]) and torch.equal(one[2], got[i])


@pytest.mark.parametrize("fmt", FORMATS)
def test_steps_that_share(model, fmt):
    """Forks' steps with their common pages taken once: close to the steps without, the same bits in
    any company."""
    cache = _cache(pages=400, dtype=fmt)
    doc, other = model.prefill_batch(_prompts([530, 70]), cache)[0]
    forks = cache.fork([doc], 5)
    again = cache.fork(forks[:4])                                # the same rows: what is taken together stays so
    plan = cache.shared([*forks, other], CFG["heads"])
    assert plan.members == [5, 1] and plan.longest == 512
    pair = cache.shared([again[2], again[0]], CFG["heads"])
    alone = cache.fork(forks)
    for t in range(18):                                          # past the end of a page
        toks = _tok(1 + t, 2, 3, 4, 5, 6)
        got = model.step_batch(toks, cache, [*forks, other], shared=plan)
        _close(got[:5], model.step_batch(toks[:5], cache, alone))
        assert torch.equal(model.step_batch(toks[[2, 0]], cache, [again[2], again[0]], shared=pair), got[[2, 0]])
    lengths = [cache.length(s) for s in forks]
    with pytest.raises(ValueError):
        model.step_batch(_tok(1, 2, 3), cache, forks[:3], shared=plan)   # another batch's
    assert [cache.length(s) for s in forks] == lengths
    cache.free([doc, other, *forks, *again, *alone])
    assert cache.free_pages == 400


@pytest.mark.parametrize("fmt", FORMATS[1:])
def test_a_failed_call_gives_its_pages_back(model, fmt):
    cache = _cache(pages=8, dtype=fmt)
    (s,), _ = model.prefill_batch(_prompts([16]), cache)
    f, = cache.fork([s])
    cache.compact([f], 3, [[]])                                 # its next row lies in a shared page
    free = cache.free_pages
    for fail in (lambda: model.step_batch(torch.tensor([1, 2]), cache, [s, f]),         # tokens on the CPU
                 lambda: model.append_batch([x.cpu() for x in _prompts([20, 30])], cache, [s, f])):
        with pytest.raises(RuntimeError):
            fail()
        assert cache.free_pages == free and cache.length(s) == 16 and cache.length(f) == 3
    with pytest.raises(RuntimeError):
        model.append_batch(_prompts([200]), cache, [s])          # too few pages
    for prompts, seqs in (([], []), (_prompts([3]), [s, f]), (_prompts([3, 0]), [s, f]), (_prompts([3, 3]), [s, s]),
                          (_prompts([3]), [99])):
        with pytest.raises(ValueError):
            model.append_batch(prompts, cache, seqs)
    assert cache.free_pages == free
    a = model.append_batch(_prompts([20, 30], 7), cache, [s, f])
    other = _cache(dtype=fmt)
    p, = _prompts([16])
    seqs, _ = model.prefill_batch([p, p[:3]], other)
    assert torch.equal(model.append_batch(_prompts([20, 30], 7), other, seqs), a)


def test_questions_about_a_document(model):
    """All of it as the documentation shows it: a document held in 8 bits, questions appended to its
    forks, answers token by token with the document's rows read once for all, scored; in the end every
    page is free."""
    from respect_amd.decoding.acceptance import greedy_token
    from respect_amd.decoding.logprobs import token_logprobs
    cache = _cache(pages=400, dtype="mxfp8")
    (doc,), _ = model.prefill_batch(_prompts([1000]), cache)
    questions = _prompts([12, 5, 30, 8], 2)
    seqs = cache.fork([doc], 4)
    logits = model.append_batch(questions, cache, seqs)
    plan = cache.shared(seqs, CFG["heads"])
    assert plan.members == [4] and plan.longest == 960
    plain = cache.fork(seqs)
    other = logits
    for _ in range(4):
        tokens = greedy_token(logits)
        given = token_logprobs(logits, tokens)[0]
        assert given.shape == (4,) and torch.isfinite(given).all()
        logits = model.step_batch(tokens, cache, seqs, shared=plan)
        other = model.step_batch(tokens, cache, plain)
        _close(logits, other)
    cache.free([doc, *seqs, *plain])
    assert cache.free_pages == 400


@pytest.mark.parametrize("fmt", FORMATS)
def test_two_streams_at_once(model, fmt):
    """Appended tokens and shared steps of two groups, enqueued on two streams behind work that holds
    both back: the bits of the same calls one after the other."""
    def start():
        cache = _cache(pages=600, dtype=fmt)
        docs, _ = model.prefill_batch(_prompts([300, 700]), cache)
        seqs = [cache.fork([d], 3) for d in docs]
        return cache, seqs, [cache.shared(s, CFG["heads"]) for s in seqs]

    def calls(cache, seqs, plans, which, step):
        if step == 0:
            return model.append_batch(_prompts([20, 3, 70], which), cache, seqs[which])
        return model.step_batch(_tok(step, which, 7), cache, seqs[which], shared=plans[which])
    state = start()
    want = [[calls(*state, w, i) for w in (0, 1)] for i in range(5)]
    state = start()
    a = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(8):
                torch.mm(a, a)
    got = []
    for i in range(5):
        got.append([])
        for w in (0, 1):
            with torch.cuda.stream(streams[w]):
                got[-1].append(calls(*state, w, i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g, v in zip(got, want) for x, y in zip(g, v))
