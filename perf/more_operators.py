"""Serving from a cache of few bits, and sharing a long beginning, as cases that can be timed.

``listed()`` holds fixed cases and ``draw(rng)`` gives further ones of the same
ranges; ``prepare`` makes what a program has in hand before the call, ``run`` is
one pass, in plain torch where ``own`` is false and through the framework's
public entry points where it is true, ``exact`` the same results in 64 bits.

The cache's formats: 32 consecutive elements of a row share a power of two, a byte e
that stands for 2^(e - 127), the smallest one (and no smaller than 2^-117) that no
element outgrows; each element is a number of 8 bits ("mxfp8": e4m3, up to 448) or of
4 ("mxfp4": e2m1, up to 6, the first of two in the low half of a byte), rounded to
nearest, ties to even.

Kinds of a case:
  store     K and V rows written to a layer's pools in such a format, and read back as
            the bf16 values that the codes stand for
  read      the rows of several sequences read back from scattered pages
  token     attention of one new token per sequence over a paged cache in such a format
  shared    the same for groups of sequences that begin with the same keys, the cache
            in such a format or in bf16
"""
import math
import random

import torch

own = False

BF = torch.bfloat16
DEV = "cuda"
HEADS_8B = {"heads": 32, "kv_heads": 8, "head_dim": 128}
BITS = {"mxfp8": 8, "mxfp4": 4}


def listed():
    return [
        # The new rows of a full batch's step in one layer: the smallest call, where latency counts.
        {"name": "store_step", "kind": "store", "tokens": 64, "page": 64, "format": "mxfp8", **HEADS_8B},
        # The rows of several packed prompts in one layer.
        {"name": "store_prompts", "kind": "store", "tokens": 16301, "page": 32, "format": "mxfp4", **HEADS_8B},
        # A few conversations continued: their earlier rows, small heads.
        {"name": "read_chunks", "kind": "read", "sequences": 5, "longest": 2500, "page": 16, "format": "mxfp8",
         "heads": 16, "kv_heads": 2, "head_dim": 64},
        # Questions about long documents that are held already.
        {"name": "read_long", "kind": "read", "sequences": 3, "longest": 100003, "page": 64, "format": "mxfp4", **HEADS_8B},
        # One user's next token some thousand tokens into a conversation.
        {"name": "token8_one", "kind": "token", "sequences": 1, "longest": 4097, "page": 16, "format": "mxfp8", **HEADS_8B},
        # A full batch in mid-answer.
        {"name": "token8_batch", "kind": "token", "sequences": 64, "longest": 8000, "page": 64, "format": "mxfp8", **HEADS_8B},
        # A small model's batch.
        {"name": "token4_batch", "kind": "token", "sequences": 48, "longest": 4001, "page": 32, "format": "mxfp4",
         "heads": 16, "kv_heads": 2, "head_dim": 64},
        # A few sequences, one with a very long cache: little to share out but the cache itself.
        {"name": "token4_long", "kind": "token", "sequences": 6, "longest": 131072, "page": 32, "format": "mxfp4", **HEADS_8B},
        # Several answers sampled for one prompt.
        {"name": "shared_few", "kind": "shared", "groups": 1, "members": 4, "longest": 2512, "tail": 200, "page": 16,
         "format": "bf16", **HEADS_8B},
        # A full batch behind one long instruction.
        {"name": "shared_batch", "kind": "shared", "groups": 1, "members": 64, "longest": 8000, "tail": 500, "page": 64,
         "format": "bf16", **HEADS_8B},
        # Several prompts, each answered several times.
        {"name": "shared_groups", "kind": "shared", "groups": 8, "members": 8, "longest": 4000, "tail": 700, "page": 32,
         "format": "mxfp8", **HEADS_8B},
        # Many questions about one very long document.
        {"name": "shared_long", "kind": "shared", "groups": 1, "members": 24, "longest": 100032, "tail": 1000, "page": 64,
         "format": "mxfp4", **HEADS_8B},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "read"] + ["token"] * 3 + ["shared"] * 3)
    h, hk, d = rng.choice([(32, 8, 128)] * 2 + [(16, 8, 128), (32, 4, 128), (8, 2, 64), (16, 2, 64)])
    case = {"kind": kind, "page": rng.choice([16, 32, 64, 128]), "format": rng.choice(["mxfp8", "mxfp4"]),
            "heads": h, "kv_heads": hk, "head_dim": d}
    if kind == "store":
        case["tokens"] = _log(rng, 1, 16000)
    elif kind == "read":
        case["sequences"] = _log(rng, 1, 64)
        case["longest"] = _log(rng, 1, 100000 // case["sequences"])
    elif kind == "token":
        case["sequences"] = _log(rng, 1, 256)
        case["longest"] = _log(rng, 1, min(131072, 786432 // case["sequences"]))
    else:
        case["format"] = rng.choice(["bf16", "bf16", "mxfp8", "mxfp4"])
        case["groups"] = _log(rng, 1, 16)
        case["members"] = _log(rng, 1, 64)
        many = case["groups"] * case["members"]
        case["longest"] = _log(rng, 50, min(100000, 2400000 // many, 400000 // case["groups"]))
        case["tail"] = _log(rng, 1, min(2000, 200000 // many))
    return case


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV).to(BF)


def _channels(g, case):
    """Keys have channels much larger than others; values have not."""
    return torch.exp(0.5 * torch.randn(case["head_dim"], generator=g, device=DEV))


def _spread(key, longest, many):
    """``many`` lengths, a function of ``key`` alone: the first one the longest, the others spread
    over the logarithm below it."""
    rng = random.Random(key)
    return [longest] + [_log(rng, 1, longest) for _ in range(many - 1)]


def _lengths(case):
    """(lengths, shared keys of each group, sequences of each group)."""
    page = case["page"]
    if case["kind"] != "shared":
        return _spread(f"{case['kind']} {case['longest']}", case["longest"], case["sequences"]), [], []
    shared = [n // page * page for n in _spread(f"shared {case['longest']}", case["longest"], case["groups"])]
    tails = _spread(f"tails {case['tail']}", case["tail"], case["groups"] * case["members"])
    return [shared[i // case["members"]] + n for i, n in enumerate(tails)], shared, [case["members"]] * case["groups"]


def _quantise(x, fmt):
    """Rows [..., D] -> (codes uint8 [..., D * bits / 8], scales uint8 [..., D / 32])."""
    g = x.float().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    frac, exp = torch.frexp(top)                       # top = frac 2^exp, frac in [0.5, 1)
    e = exp - 9 + (frac > 0.875) if fmt == "mxfp8" else exp - 3 + (frac > 0.75)
    e = torch.where(top == 0, -117, e).clamp(min=-117)
    y = (torch.ldexp(g, -e)).flatten(-2)
    if fmt == "mxfp8":
        codes = y.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = y.abs()
        n = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)) + 8 * torch.signbit(y)
        n = n.to(torch.uint8).unflatten(-1, (-1, 2))
        codes = n[..., 0] | n[..., 1] << 4
    return codes, (e[..., 0] + 127).to(torch.uint8)


def _values(codes, scales, fmt):
    """The fp32 values of rows of codes."""
    if fmt == "mxfp8":
        y = codes.view(torch.float8_e4m3fn).float()
    else:
        half = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
        n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
        y = half[n & 7] * (1 - 2.0 * (n >> 3))
    return torch.ldexp(y.unflatten(-1, (-1, 32)), scales.int()[..., None] - 127).flatten(-2)


def _pools(case, slots, g):
    """One layer's K and V pools: bf16 [HK, slots, D], or (codes, scales) of it."""
    out, chan = [], _channels(g, case)
    for side in range(2):
        heads = []
        for _ in range(case["kv_heads"]):
            x = torch.randn(slots, case["head_dim"], generator=g, device=DEV) * (chan if side == 0 else 1.0)
            heads.append(x.to(BF) if case["format"] == "bf16" else _quantise(x.to(BF), case["format"]))
        out.append(torch.stack(heads) if case["format"] == "bf16" else tuple(torch.stack(t) for t in zip(*heads)))
    return out


def _tables(case, g):
    """(table [B, width], lens, slots): pages in no order, as after some time of serving, with a few
    free ones between them; a group's sequences hold the pages of their common beginning together."""
    lens, shared, members = _lengths(case)
    page = case["page"]
    used = [-(-n // page) for n in lens]
    common = [n // page for n, m in zip(shared, members) for _ in range(m)] or [0] * len(lens)
    pages = sum(used) - sum(common) + sum(n // page for n in shared) + 3
    order = torch.randperm(pages, generator=g, device=DEV).cpu()
    table = torch.zeros(len(lens), max(used), dtype=torch.int32)
    at, b = 0, 0
    for n, m in zip(shared, members):
        table[b:b + m, :n // page] = order[at:at + n // page]
        at, b = at + n // page, b + m
    for i, n in enumerate(used):
        table[i, common[i]:n] = order[at:at + n - common[i]]
        at += n - common[i]
    return table, lens, pages * page


def _store_inputs(case, seed):
    g, n, page = _gen(seed), case["tokens"], case["page"]
    shape = (n, case["kv_heads"], case["head_dim"])
    k = (torch.randn(*shape, generator=g, device=DEV) * _channels(g, case)).to(BF)
    v = _randn(g, *shape)
    # A step's rows lie in as many pages; a prompt's fill theirs.
    pages = n + 3 if n <= 256 else -(-n // page) + 3
    order = torch.randperm(pages, generator=g, device=DEV)
    j = torch.arange(n, device=DEV)
    slots = order * page + torch.randint(0, page, (pages,), generator=g, device=DEV) if n <= 256 else None
    slots = slots[:n] if n <= 256 else order[j // page] * page + j % page
    return [k, v, slots.to(torch.int32), pages * page]


def _read_inputs(case, seed):
    g = _gen(seed)
    table, lens, slots = _tables(case, g)
    pools = _pools(case, slots, g)
    rows = []
    for t, n in zip(table, lens):
        j = torch.arange(n)
        rows.append(t[j // case["page"]] * case["page"] + j % case["page"])
    return [*pools, torch.cat(rows).to(torch.int32).to(DEV), slots]


def _attn_inputs(case, seed):
    g = _gen(seed)
    table, lens, slots = _tables(case, g)
    q = _randn(g, len(lens), case["heads"], case["head_dim"])
    return [q, *_pools(case, slots, g), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), lens]


def _own_rows(pool, fmt):
    from respect_amd.kernels.mx import MXRows
    return pool if fmt == "bf16" else MXRows(*pool, fmt)


def prepare(case, seed):
    kind, fmt = case["kind"], case["format"]
    if kind in ("store", "read"):
        a = _store_inputs(case, seed) if kind == "store" else _read_inputs(case, seed)
        slots = a.pop()
        if not own:
            if kind == "store":
                D, HK = case["head_dim"], case["kv_heads"]
                a += [tuple(torch.zeros(HK, slots, n, dtype=torch.uint8, device=DEV) for n in (D * BITS[fmt] // 8, D // 32))
                      for _ in range(2)]
            return case, a
        from respect_amd.decoding.paged_kv import PagedKVCache
        cache = PagedKVCache(1, case["kv_heads"], case["head_dim"], slots // case["page"], page=case["page"], device=DEV,
                             dtype=fmt)
        if kind == "read":
            for mine, (codes, scales) in ((cache.k[0], a.pop(0)), (cache.v[0], a.pop(0))):
                mine.codes.copy_(codes)
                mine.scales.copy_(scales)
        return case, [cache, *a]
    q, kc, vc, table, lens, counts = _attn_inputs(case, seed)
    if not own:
        return case, [q, kc, vc, table, counts]
    a = [q, _own_rows(kc, fmt), _own_rows(vc, fmt), table, lens]
    if kind == "shared":
        from respect_amd.kernels.paged_attention import SharedPrefix
        _, shared, members = _lengths(case)
        a.append(SharedPrefix(members, shared, case["heads"] // case["kv_heads"], device=DEV))
    return case, a


# ------------------------------------------------------------------ one pass

def run(state):
    return _run_own(*state) if own else _run_plain(*state)


def _run_own(case, a):
    kind = case["kind"]
    if kind == "store":
        cache, k, v, slots = a
        cache.write(0, k, v, slots)
        return cache.read(0, slots)
    if kind == "read":
        cache, slots = a
        return cache.read(0, slots)
    from respect_amd.kernels.paged_attention import paged_attn
    q, kc, vc, table, lens, *plan = a
    return paged_attn(q, kc, vc, table, lens, case["page"], shared=plan[0] if plan else None)


def _run_plain(case, a):
    kind, fmt = case["kind"], case["format"]
    if kind == "store":
        k, v, slots, *pools = a
        for x, (codes, scales) in zip((k, v), pools):
            c, s = _quantise(x, fmt)
            codes[:, slots.long()], scales[:, slots.long()] = c.transpose(0, 1), s.transpose(0, 1)
        return [_gather(p, slots.long(), fmt).transpose(0, 1).to(BF) for p in pools]
    if kind == "read":
        *pools, slots = a
        return [_gather(p, slots.long(), fmt).transpose(0, 1).to(BF) for p in pools]
    return _plain_attn(case, *a)


def _gather(pool, slots, fmt):
    """fp32 rows [HK, n, D] of a pool."""
    if fmt == "bf16":
        return pool[:, slots].float()
    return _values(pool[0][:, slots], pool[1][:, slots], fmt)


def _plain_attn(case, q, kc, vc, table, counts):
    B, H, D = q.shape
    HK, page = case["kv_heads"], case["page"]
    out = torch.empty_like(q)
    for b, n in enumerate(counts):
        j = torch.arange(n, device=DEV)
        slots = table[b, j // page].long() * page + j % page
        ks, vs = (_gather(x, slots, case["format"]) for x in (kc, vc))
        s = q[b].float().view(HK, H // HK, D) @ ks.transpose(1, 2).contiguous() * D ** -0.5
        e = torch.exp(s - s.amax(-1, keepdim=True))
        out[b] = (e / e.sum(-1, keepdim=True) @ vs).view(H, D).to(BF)
    return out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind, D, HK = case["kind"], case["head_dim"], case["kv_heads"]
    row = 4 * D if case["format"] == "bf16" else 2 * (D * BITS[case["format"]] // 8 + D // 32)   # K and V of a head
    if kind == "store":
        return {"bytes": case["tokens"] * (HK * (8 * D + row) + 4), "flops": 4 * case["tokens"] * HK * D}
    lens, shared, members = _lengths(case)
    if kind == "read":
        return {"bytes": sum(lens) * (HK * (4 * D + row) + 4), "flops": 2 * sum(lens) * HK * D}
    keys = sum(lens) - sum(n * (m - 1) for n, m in zip(shared, members))
    table = 4 * sum(-(-n // case["page"]) for n in lens)
    return {"bytes": keys * HK * row + 4 * D * case["heads"] * len(lens) + table, "flops": 4 * case["heads"] * D * sum(lens)}


# ------------------------------------------------------------------ 64-bit results

def _table64(fmt):
    """The value of every code, from the formats' definition."""
    bits, mant, bias = (8, 3, 7) if fmt == "mxfp8" else (4, 1, 1)
    out = []
    for c in range(1 << bits):
        m, e = c & (1 << mant) - 1, c >> mant & (1 << bits - 1 - mant) - 1
        x = math.ldexp(m, 1 - bias - mant) if e == 0 else math.ldexp(m + (1 << mant), e - bias - mant)
        out.append(-x if c >> bits - 1 else x)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _rows64(pool, h, slots, case):
    """Rows ``slots`` of head h in 64 bits."""
    if case["format"] == "bf16":
        return pool[h, slots].double()
    c, s = pool[0][h, slots].long(), pool[1][h, slots].double()
    if case["format"] == "mxfp4":
        c = torch.stack((c % 16, c // 16), 2).reshape(len(c), -1)
    return _table64(case["format"])[c] * torch.exp2(s - 127).repeat_interleave(32, 1)


def _stored64(x, fmt):
    x = x.double()
    most, mant, low = (448.0, 3, -6) if fmt == "mxfp8" else (6.0, 1, 0)
    groups = x.reshape(*x.shape[:-1], -1, 32)
    top = groups.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(top / most)).clamp(min=-117.0))
    scale = torch.where(top > most * scale, 2 * scale, scale)               # where log2's rounding misled
    scale = torch.where((top <= most * scale / 2) & (scale > 2.0 ** -117), scale / 2, scale)
    y = groups / scale
    step = torch.exp2(torch.frexp(y)[1].double().sub(1).clamp(min=low) - mant)
    return (torch.round(y / step) * step * scale).reshape(x.shape)


def exact(case, seed):
    kind, fmt = case["kind"], case["format"]
    HK, G, D, page = case["kv_heads"], case["heads"] // case["kv_heads"], case["head_dim"], case["page"]
    if kind == "store":
        k, v, _, _ = _store_inputs(case, seed)
        return [_stored64(k, fmt), _stored64(v, fmt)]
    if kind == "read":
        *pools, slots, _ = _read_inputs(case, seed)
        return [torch.stack([_rows64(p, h, slots.long(), case) for h in range(HK)], 1) for p in pools]
    q, kc, vc, table, _, counts = _attn_inputs(case, seed)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(counts):
        slots = (table[b, :-(-n // page), None].long() * page + torch.arange(page, device=DEV)).view(-1)[:n]
        for h in range(HK):
            s = _rows64(kc, h, slots, case) @ q[b, h * G:(h + 1) * G].double().t() * D ** -0.5
            out[b, h * G:(h + 1) * G] = torch.softmax(s, 0).t() @ _rows64(vc, h, slots, case)
    return out
