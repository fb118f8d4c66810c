"""The microscaled formats of a cache's rows from their definition, in 64 bits on the CPU."""
import torch

BITS = {"mxfp8": 8, "mxfp4": 4}
# The codes without a sign in the order of their values: e4m3 (127 is its NaN), e2m1.
POSITIVE = {"mxfp8": [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
            "mxfp4": [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]}


def quantise(x, fmt):
    """bf16 rows [..., D] -> (codes [..., D * bits / 8], scales [..., D / 32]) uint8."""
    v = torch.tensor(POSITIVE[fmt], dtype=torch.float64)
    g = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    a = torch.where(bad, 0.0, g.abs())
    e = torch.full(bad.shape, -117, dtype=torch.int32)
    top = a.amax(-1, keepdim=True)
    for s in range(-116, 129):                           # the smallest that no element outgrows
        e = torch.where(top > v[-1] * 2.0 ** (s - 1), s, e)
    y = a / 2.0 ** e.double()
    hi = torch.searchsorted(v, y).clamp(max=len(v) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = v[hi] - y, y - v[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(y == v[hi], hi, code) | (torch.signbit(x.double()).unflatten(-1, (-1, 32)).long() << (BITS[fmt] - 1))
    code = torch.where(bad, 0, code).flatten(-2).to(torch.uint8)
    if fmt == "mxfp4":
        code = code[..., ::2] | code[..., 1::2] << 4
    return code.contiguous(), torch.where(bad, 255, e + 127)[..., 0].to(torch.uint8)


def values(codes, scales, fmt):
    """float64 values of rows of codes."""
    v = torch.tensor(POSITIVE[fmt] + [float("nan")] * (fmt == "mxfp8"), dtype=torch.float64)
    table = torch.cat((v, -v))
    if fmt == "mxfp4":
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    s = torch.where(scales == 255, float("nan"), 2.0 ** (scales.double() - 127))
    return (table[codes.long()].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)
