"""Pools whose slot offsets alone, and whose head offsets alone, pass 2^32 bytes: rows written, read and
moved, attention with a plan and without, against pools that lie together.  A product cut to 32 bits
would land on other rows of the same memory."""
import pytest
import torch

from test_mx_rows import _same
from test_shared_attention import BF, FORMATS, _cache, _i32, _plan, _q

pytestmark = pytest.mark.gpu

PAGE, PAGES, PITCH = 16, 272, 1 << 20      # bytes from slot to slot


def _wide():
    """Zeros [2, slots, PITCH] in which both kinds of offset pass 32 bits."""
    base = torch.zeros(2, PAGES * PAGE, PITCH, dtype=torch.uint8, device="cuda")
    assert base.stride(0) > 1 << 32 and (PAGES - 12) * PAGE * base.stride(1) > 1 << 32 and base.stride(1) < 1 << 31
    return base


def _at(base, n, column, dtype=torch.uint8):
    """Rows of n elements from byte ``column`` of every slot on."""
    x = base.view(dtype)
    size = torch.empty(0, dtype=dtype).element_size()
    return x[:, :, column // size:column // size + n]


def _place(i):
    """Page i of a small pool: the last and the first pages of the wide one in turn."""
    return i // 2 if i % 2 else PAGES - 1 - i // 2


def _spread(base, small, fmt, columns):
    """The rows of a small pool in the wide one; (codes or rows, scales) from ``columns`` on."""
    from respect_amd.kernels.mx import MXRows
    parts = [small] if fmt == "bf16" else [small.codes, small.scales]
    out = []
    for p, c in zip(parts, columns):
        x = _at(base, p.shape[2], c, p.dtype)
        n = p.shape[1] // PAGE
        assert n <= 24
        x.view(2, PAGES, PAGE, -1)[:, [_place(i) for i in range(n)]] = p.view(2, n, PAGE, -1)
        out.append(x)
    return out[0] if fmt == "bf16" else MXRows(*out, fmt)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fmt", FORMATS)
def test_attention(fmt, D):
    from respect_amd.kernels.paged_attention import paged_attn
    members, keys, lens = [3], [64], [64, 100, 90]
    kc, vc, table, _ = _cache(lens, PAGE, 2, D, fmt, members, keys, seed=2)
    base, new = _wide(), table.clone()
    for i in range(table.numel()):
        if table.view(-1)[i] >= 0:
            new.view(-1)[i] = _place(int(table.view(-1)[i]))
    assert (new >= PAGES - 12).any() and ((new >= 0) & (new < 12)).any()
    k2, v2 = _spread(base, kc, fmt, (0, 4096)), _spread(base, vc, fmt, (32768, 65536 + 2))
    q = _q(3, 8, D).cuda()
    for plan in (_plan(members, keys, 4), None):
        want = paged_attn(q, kc, vc, table.cuda(), _i32(lens), PAGE, shared=plan)
        assert torch.isfinite(want.float()).all()
        assert torch.equal(paged_attn(q, k2, v2, new.cuda(), _i32(lens), PAGE, shared=plan), want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows(fmt):
    """Written (few bits), read, and moved in lists of either kind."""
    from respect_amd import _lib
    from respect_amd.kernels.mx import BITS, MXRows, read_rows, write_rows
    D, base = 64, _wide()
    slots = [PAGES * PAGE - 1, 0, 4100, 4097, 17, 4300]
    assert sum(s * PITCH > 1 << 32 for s in slots) == 4
    x = torch.randn(len(slots), 2, D, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    y = x.flip(0).contiguous()
    if fmt == "bf16":
        k, v = _at(base, D, 0, BF), _at(base, D, 4096, BF)
        for i, s in enumerate(slots):
            k[:, s], v[:, s] = x[i], y[i]
        want = x, y
    else:
        n = D * BITS[fmt] // 8
        k = MXRows(_at(base, n, 0), _at(base, 2, 8192), fmt)
        v = MXRows(_at(base, n, 4096), _at(base, 2, 8192 + 2), fmt)
        small = [MXRows.empty(2, 6, D, fmt) for _ in range(2)]
        write_rows(x, y, *small, _i32(range(6)))
        write_rows(x, y, k, v, _i32(slots))
        want = read_rows(*small, _i32(range(6)))
        for a, b in ((k, small[0]), (v, small[1])):
            assert torch.equal(a.codes[:, slots], b.codes) and torch.equal(a.scales[:, slots], b.scales)
        assert int((base != 0).sum()) == sum(int((t != 0).sum()) for p in small for t in (p.codes, p.scales))
    assert all(_same(a, b) for a, b in zip(read_rows(k, v, _i32(slots)), want))
    moves = [(s, t) for s, t in zip(slots, (4101, 4351 - 8, 1, 4200, 4201, 2))]
    groups, flat = [0, 2, 6], [n for m in moves for n in m]
    L = _lib.lib()
    parts = [k, v] if fmt == "bf16" else [k.codes, v.codes, k.scales, v.scales]
    bases = torch.tensor([p.data_ptr() for p in parts], device="cuda")
    sh, sn = parts[0].stride(0), parts[0].stride(1)
    for on_host in (True, False):
        lists = torch.tensor(groups + flat, dtype=torch.int32, device="cpu" if on_host else "cuda")
        at = lists.data_ptr(), 2, lists.data_ptr() + 12, 6
        stream = _lib.stream_ptr(bases.device)
        if fmt == "bf16":
            fn = L.rspx_kv_move_values if on_host else L.rspx_kv_move
            rc = fn(bases.data_ptr(), 2, 2, D, sh, sn, PAGES * PAGE, *at, stream)
        else:
            fn = L.rspx_kv_move_mx_values if on_host else L.rspx_kv_move_mx
            rc = fn(bases.data_ptr(), 2, 2, D, BITS[fmt], sh, sn, parts[2].stride(0), parts[2].stride(1), PAGES * PAGE, *at, stream)
        assert rc == 0
        to = _i32([t for _, t in moves])
        assert all(_same(a, b) for a, b in zip(read_rows(k, v, to), want))
        for p in parts:
            p[:, to.long()] = 0
