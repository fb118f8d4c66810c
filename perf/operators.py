"""Serving several requests at once, as cases that can be timed.

``listed()`` holds fixed cases and ``draw(rng)`` gives further ones of the same
ranges; ``prepare`` makes what a program has in hand before the call, ``run`` is
one pass, in plain torch where ``own`` is false and through the framework's
public entry points where it is true, ``exact`` the same results in 64 bits.

Kinds of a case:
  prompt    causal attention over whole prompts of different lengths, packed one
            after the other; ``earlier`` keys before each prompt's own
  token     attention of one new token per sequence over a paged KV cache
  fork      sequences of a paged cache forked ``copies`` times each (full pages
            shared, the begun page's rows copied in every layer), their tables
            made, and the forks freed again
  compact   the accepted path of a verified trie moved to consecutive rows of its
            sequence, all layers and sequences at once, and room made for the
            next trie
  logprobs  log probabilities of given tokens, entropy and the best alternatives
"""
import math
import random

import numpy as np
import torch

own = False

BF = torch.bfloat16
DEV = "cuda"
HEADS_8B = {"heads": 32, "kv_heads": 8, "head_dim": 128}
VOCAB = 151936


def listed():
    return [
        # One short question: the smallest prompt, where latency counts.
        {"name": "prompt_short", "kind": "prompt", "sequences": 1, "longest": 77, "earlier": 0, **HEADS_8B},
        # A batch of prompts of very different lengths, from a few tokens to some thousand.
        {"name": "prompt_packed", "kind": "prompt", "sequences": 24, "longest": 4099, "earlier": 0, **HEADS_8B},
        # A few prompts that continue a long common beginning, small heads.
        {"name": "prompt_chunks", "kind": "prompt", "sequences": 5, "longest": 1021, "earlier": 2500,
         "heads": 16, "kv_heads": 2, "head_dim": 64},
        # One very long document.
        {"name": "prompt_long", "kind": "prompt", "sequences": 1, "longest": 16384, "earlier": 0, **HEADS_8B},
        # One user's next token some thousand tokens into a conversation.
        {"name": "token_one", "kind": "token", "sequences": 1, "longest": 4097, "page": 16, **HEADS_8B},
        # A full batch in mid-answer.
        {"name": "token_batch", "kind": "token", "sequences": 64, "longest": 8000, "page": 64, **HEADS_8B},
        # A few sequences, one with a very long cache: little to share out but the cache itself.
        {"name": "token_long", "kind": "token", "sequences": 6, "longest": 131072, "page": 32, **HEADS_8B},
        # Several answers sampled for one prompt.
        {"name": "fork_few", "kind": "fork", "sequences": 1, "copies": 4, "longest": 333, "page": 16, "layers": 24,
         "kv_heads": 8, "head_dim": 128},
        # The same for a batch of prompts.
        {"name": "fork_batch", "kind": "fork", "sequences": 32, "copies": 4, "longest": 500, "page": 64, "layers": 24,
         "kv_heads": 8, "head_dim": 128},
        # A batch of tries was verified and a late branch of each accepted.
        {"name": "compact_batch", "kind": "compact", "sequences": 32, "longest": 400, "nodes": 64, "kept": 3, "moved": 13,
         "page": 64, "layers": 24, "kv_heads": 8, "head_dim": 128},
        # One sampled token's score, and the alternatives shown beside it.
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "vocab": VOCAB, "top": 20},
        # The scores of a prompt's own tokens.
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 1500, "vocab": VOCAB, "top": 5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt"] * 3 + ["token"] * 3 + ["fork", "compact"] + ["logprobs"] * 2)
    h, hk, d = rng.choice([(32, 8, 128)] * 2 + [(16, 8, 128), (32, 4, 128), (8, 2, 64), (16, 2, 64)])
    heads = {"heads": h, "kv_heads": hk, "head_dim": d}
    if kind == "prompt":
        n = _log(rng, 1, 32)
        earlier = rng.choice([0, 0, _log(rng, 1, 4096)])
        return {"kind": kind, "sequences": n, "longest": _log(rng, 1, (2048 if earlier else 16384) / math.sqrt(n)),
                "earlier": earlier, **heads}
    if kind == "token":
        n = _log(rng, 1, 256)
        return {"kind": kind, "sequences": n, "longest": _log(rng, 1, min(131072, 786432 // n)),
                "page": rng.choice([16, 32, 64, 128]), **heads}
    if kind == "logprobs":
        vocab = rng.choice([VOCAB, VOCAB, _log(rng, 50, VOCAB)])
        return {"kind": kind, "rows": _log(rng, 1, 1500), "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 50])}
    case = {"kind": kind, "sequences": _log(rng, 1, 32), "longest": _log(rng, 1, 500),
            "page": rng.choice([16, 32, 64]), "layers": _log(rng, 1, 24), "kv_heads": hk, "head_dim": d}
    if kind == "fork":
        case["copies"] = rng.randint(1, 4)
    else:
        case["kept"], case["moved"] = rng.randint(0, 6), rng.randint(1, 24)
        case["nodes"] = case["kept"] + 2 * case["moved"] + rng.randint(0, 20)
    return case


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(BF)


def _lengths(case):
    """The sequences' lengths: a function of the case alone, the first one the longest and the
    others spread over the logarithm below it."""
    rng = random.Random(f"{case['kind']} {case['sequences']} {case['longest']}")
    return [case["longest"]] + [_log(rng, 1, case["longest"]) for _ in range(case["sequences"] - 1)]


def _prompt_inputs(case, seed):
    g = _gen(seed)
    rows = _lengths(case)
    keys = [n + case["earlier"] for n in rows]
    H, HK, D = case["heads"], case["kv_heads"], case["head_dim"]
    # Normalised q and k (unit elements; a score's scale is D ** -0.5) and v of unit scale.
    q = _randn(g, sum(rows), H, D)
    k, v = _randn(g, sum(keys), HK, D), _randn(g, sum(keys), HK, D)
    return [q, k, v, rows, keys]


def _token_inputs(case, seed):
    g = _gen(seed)
    lens, page = _lengths(case), case["page"]
    H, HK, D = case["heads"], case["kv_heads"], case["head_dim"]
    q = _randn(g, len(lens), H, D)
    used = [-(-n // page) for n in lens]
    # Pages in no order, as after some time of serving, with a few free ones between them.
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device=DEV).cpu().tolist()
    table = torch.zeros(len(lens), max(used), dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    kc, vc = (torch.empty(HK, pages * page, D, dtype=BF, device=DEV) for _ in range(2))
    for t in (kc, vc):
        for h in range(HK):
            t[h] = _randn(g, pages * page, D)
    return [q, kc, vc, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), lens]


def _pages_needed(case):
    extra = case.get("nodes", 0)
    return sum(-(-(n + extra) // case["page"]) for n in _lengths(case))


def _pool(case, seed):
    """K and V pools per layer of a cache whose sequences take the lowest pages in turn."""
    g = _gen(seed)
    spare = case["sequences"] * case.get("copies", 0) + 2
    slots = (_pages_needed(case) + spare) * case["page"]
    shape = (case["kv_heads"], slots, case["head_dim"])
    return [[_randn(g, *shape) for _ in range(case["layers"])] for _ in range(2)]


def _path(case):
    """Accepted nodes: the first ``kept`` ones, then the end of a branch inserted later."""
    first = case["nodes"] - case["moved"]
    return list(range(case["kept"])) + list(range(first, case["nodes"]))


def _logits(case, seed):
    g = _gen(seed)
    # Scores as a vocabulary projection leaves them: a broad bulk, a few likely tokens.
    x = torch.randn(case["rows"], case["vocab"], generator=g, device=DEV) * 2.5
    tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device=DEV)
    x[torch.arange(case["rows"], device=DEV), tokens] += 12.0
    return [x, tokens]


class _PlainPages:
    """The page bookkeeping of a cache on the host: who holds which page, lowest page first."""

    def __init__(self, case):
        self.page = case["page"]
        self.lens, self.tables, at = _lengths(case), [], 0
        for n in self.lens:
            m = -(-(n + case.get("nodes", 0)) // self.page)
            self.tables.append(list(range(at, at + m)))
            at += m
        self.first_free = at


def _own_pages(case, pool):
    from respect_amd.decoding.paged_kv import PagedKVCache
    extra = case.get("nodes", 0)
    cache = PagedKVCache(case["layers"], case["kv_heads"], case["head_dim"], pool[0][0].shape[1] // case["page"],
                         page=case["page"], device=DEV)
    for mine, given in ((cache.k, pool[0]), (cache.v, pool[1])):
        for a, b in zip(mine, given):
            a.copy_(b)
    seqs = cache.add([n + extra for n in _lengths(case)])
    return cache, seqs


def prepare(case, seed):
    kind = case["kind"]
    if kind == "prompt":
        q, k, v, rows, keys = _prompt_inputs(case, seed)
        if own:
            from respect_amd.kernels.prompt_attention import PackedPrompts
            return case, [q, k, v, PackedPrompts(rows, keys, device=DEV)]
        return case, [q, k, v, rows, keys]
    if kind == "token":
        return case, _token_inputs(case, seed)
    if kind == "logprobs":
        return case, _logits(case, seed)
    pool = _pool(case, seed)
    return case, list(_own_pages(case, pool)) if own else [pool, _PlainPages(case)]


# ------------------------------------------------------------------ one pass

def run(state):
    return _run_own(*state) if own else _run_plain(*state)


def _run_own(case, a):
    kind = case["kind"]
    if kind == "prompt":
        from respect_amd.kernels.prompt_attention import prompt_attn
        return prompt_attn(*a)
    if kind == "token":
        from respect_amd.kernels.paged_attention import paged_attn
        q, kc, vc, table, lens, _ = a
        return paged_attn(q, kc, vc, table, lens, case["page"])
    if kind == "logprobs":
        from respect_amd.decoding.logprobs import token_logprobs
        return token_logprobs(*a, top=case["top"])
    cache, seqs = a
    if kind == "fork":
        forks = cache.fork(seqs, case["copies"])
        table, lens = cache.tables(forks)
        cache.free(forks)
        return [table, lens] + cache.k + cache.v
    path = _path(case)
    cache.compact(seqs, _lengths(case), [path] * len(seqs))
    table, lens = cache.tables(seqs)
    cache.extend(seqs, case["nodes"] - len(path))
    return [table, lens] + cache.k + cache.v


def _run_plain(case, a):
    kind = case["kind"]
    if kind == "prompt":
        return _plain_prompt(*a)
    if kind == "token":
        return _plain_token(case, *a)
    if kind == "logprobs":
        return _plain_logprobs(case, *a)
    return _plain_fork(case, *a) if kind == "fork" else _plain_compact(case, *a)


def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_prompt(q, k, v, rows, keys):
    T, H, D = q.shape
    HK = k.shape[1]
    G = H // HK
    out = torch.empty_like(q)
    t = j = 0
    for n, m in zip(rows, keys):
        closed = torch.arange(m, device=DEV)[None] > torch.arange(m - n, m, device=DEV)[:, None]
        step = max(1, min(HK, (1 << 28) // (G * n * m)))    # kv heads whose scores are held at once
        for h in range(0, HK, step):
            e = min(HK, h + step)
            qs = q[t:t + n, h * G:e * G].float().view(n, e - h, G, D).permute(1, 2, 0, 3).reshape(e - h, G * n, D)
            ks, vs = (x[j:j + m, h:e].float().transpose(0, 1).contiguous() for x in (k, v))
            s = (qs @ ks.transpose(1, 2).contiguous() * D ** -0.5).view(e - h, G, n, m)
            p = _softmax(s.masked_fill_(closed, -math.inf)).view(e - h, G * n, m)
            o = (p @ vs).view(e - h, G, n, D).permute(2, 0, 1, 3).reshape(n, (e - h) * G, D)
            out[t:t + n, h * G:e * G] = o.to(BF)
        t, j = t + n, j + m
    return out


def _plain_token(case, q, kc, vc, table, lens, counts):
    B, H, D = q.shape
    HK, page = kc.shape[0], case["page"]
    out = torch.empty_like(q)
    for b, n in enumerate(counts):
        j = torch.arange(n, device=DEV)
        slots = table[b, j // page].long() * page + j % page
        ks, vs = (x[:, slots].float() for x in (kc, vc))
        s = q[b].float().view(HK, H // HK, D) @ ks.transpose(1, 2).contiguous() * D ** -0.5
        out[b] = (_softmax(s) @ vs).view(H, D).to(BF)
    return out


def _plain_logprobs(case, x, tokens):
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = m + torch.log(z)
    given = torch.gather(x, 1, tokens[:, None]) - lse
    entropy = torch.log(z) - (e * (x - m)).sum(-1, keepdim=True) / z
    top = torch.sort(x, dim=-1, descending=True, stable=True)
    n = min(case["top"], case["vocab"])
    return [given[:, 0], entropy[:, 0], top.values[:, :n] - lse, top.indices[:, :n].contiguous()]


def _device_tables(tables, lens):
    width = max(map(len, tables))
    table = np.full((len(tables), width), -1, np.int32)
    for i, t in enumerate(tables):
        table[i, :len(t)] = t
    return torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV)


def _plain_fork(case, pool, pages):
    page, free = pages.page, pages.first_free
    tables, lens, src, dst = [], [], [], []
    for table, n in zip(pages.tables, pages.lens):
        for _ in range(case["copies"]):
            mine = list(table)
            if n % page:
                at = table[-1] * page
                src.extend(range(at, at + n % page))
                dst.extend(range(free * page, free * page + n % page))
                mine[-1], free = free, free + 1
            tables.append(mine)
            lens.append(n)
    src, dst = (torch.tensor(x, dtype=torch.int64).to(DEV) for x in (src, dst))
    for layer in pool[0] + pool[1]:
        layer[:, dst] = layer[:, src]
    return list(_device_tables(tables, lens)) + pool[0] + pool[1]


def _plain_compact(case, pool, pages):
    page, path = pages.page, _path(case)
    src, dst = [], []
    for table, n in zip(pages.tables, pages.lens):
        for i, p in enumerate(path):
            if i != p:
                src.append(table[(n + p) // page] * page + (n + p) % page)
                dst.append(table[(n + i) // page] * page + (n + i) % page)
    src, dst = (torch.tensor(x, dtype=torch.int64).to(DEV) for x in (src, dst))
    for layer in pool[0] + pool[1]:
        layer[:, dst] = layer[:, src]
    return list(_device_tables(pages.tables, [n + len(path) for n in pages.lens])) + pool[0] + pool[1]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    lens = _lengths(case)
    HK, D = case["kv_heads"], case["head_dim"]
    if kind == "prompt":
        rows, keys = sum(lens), sum(lens) + len(lens) * case["earlier"]
        pairs = sum(n * case["earlier"] + n * (n + 1) / 2 for n in lens)
        return {"bytes": 4 * D * (case["heads"] * rows + HK * keys), "flops": 4 * case["heads"] * D * pairs}
    if kind == "token":
        table = 4 * sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 4 * D * (HK * sum(lens) + case["heads"] * len(lens)) + table,
                "flops": 4 * case["heads"] * D * sum(lens)}
    row = case["layers"] * HK * D * 4     # bytes of one token's K and V in every layer
    if kind == "fork":
        rows = sum(n % case["page"] for n in lens)
        return {"bytes": row * rows * (1 + case["copies"]), "flops": 0}
    return {"bytes": 2 * row * case["sequences"] * case["moved"], "flops": 0}


# ------------------------------------------------------------------ 64-bit results

def exact(case, seed):
    kind = case["kind"]
    if kind == "prompt":
        q, k, v, rows, keys = _prompt_inputs(case, seed)
        G, scale = case["heads"] // case["kv_heads"], case["head_dim"] ** -0.5
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        t = j = 0
        for n, m in zip(rows, keys):
            for h in range(case["heads"]):
                kd, vd = k[j:j + m, h // G].double(), v[j:j + m, h // G].double()
                for r in range(0, n, 4096):
                    c = min(n, r + 4096)
                    s = q[t + r:t + c, h].double() @ kd.t() * scale
                    seen = torch.ones(c - r, m, dtype=torch.bool, device=DEV).tril(m - n + r)
                    out[t + r:t + c, h] = torch.softmax(torch.where(seen, s, -math.inf), -1) @ vd
            t, j = t + n, j + m
        return out
    if kind == "token":
        q, kc, vc, table, _, counts = _token_inputs(case, seed)
        G, page, D = case["heads"] // case["kv_heads"], case["page"], case["head_dim"]
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(counts):
            held = table[b, :-(-n // page)].long()
            for h in range(case["kv_heads"]):
                kd, vd = (x[h].view(-1, page, D)[held].view(-1, D)[:n].double() for x in (kc, vc))
                s = kd @ q[b, h * G:(h + 1) * G].double().t() * D ** -0.5
                out[b, h * G:(h + 1) * G] = torch.softmax(s, 0).t() @ vd
        return out
    if kind == "logprobs":
        x, tokens = _logits(case, seed)
        n = min(case["top"], case["vocab"])
        given, entropy, values, ids = [], [], [], []
        for r in range(0, case["rows"], 64):
            lp = torch.log_softmax(x[r:r + 64].double(), -1)
            given.append(lp.gather(1, tokens[r:r + 64, None])[:, 0])
            entropy.append(-(lp.exp() * lp).sum(-1))
            order = torch.argsort(x[r:r + 64], dim=-1, descending=True, stable=True)[:, :n]
            values.append(lp.gather(1, order))
            ids.append(order)
        return [torch.cat(given), torch.cat(entropy), torch.cat(values), torch.cat(ids)]
    return None     # rows are moved, nothing is computed
