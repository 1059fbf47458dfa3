"""Plain 64-bit forms and error bounds for the tests of the fused products.

Bounds count roundings.  u(t) is half a step of the 2-byte type.  A sum of K
products in fp32 is off by at most (K + 16) 2^-23 sum |a b|: each of at most K
accumulation steps loses at most one unit in the last place (2^-23, the tensor
core truncates) of a partial sum that is never above sum |a b|.
"""
import math

import torch

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half the smallest step


def u(t):
    return torch.finfo(t).eps / 2


def sum_err(a, b):
    """Bound of a @ b.T's error for 64-bit a (M, K), b (N, K)."""
    return (a.shape[1] + 16) * 2.0 ** -23 * (a.abs() @ b.abs().T)


def rounded(v, t):
    """Bound of rounding v once to t."""
    return v.abs() * u(t) + TINY[t]


def act64(g, act):
    """act(g) and act'(g) in 64 bits."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if act == "gelu":
        c = 0.5 * torch.special.erfc(-g / math.sqrt(2))
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * a * (g + 0.044715 * g ** 3))
    return g * s, s + g * s * (1 - s) * 2 * a * (1 + 3 * 0.044715 * g * g)


def rand(gen, t, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(t)


def framed(gen, t, rows, cols, ld_pad, offset, scale=1.0, fill=None):
    """A rows x cols matrix inside a larger buffer: row stride cols + ld_pad,
    starting `offset` elements in.  Returns (view, buffer)."""
    ld = cols + ld_pad
    buf = torch.full((offset + rows * ld + 40,), float("nan") if fill is None else fill,
                     device="cuda", dtype=t)
    view = buf[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    if fill is None:
        view.copy_(rand(gen, t, rows, cols, scale=scale))
    return view, buf


def outside_untouched(view, buf, fill):
    """Whether every element of buf outside view still holds `fill`."""
    seen = buf.clone()
    off = view.storage_offset()
    torch.as_strided(seen, view.shape, view.stride(), off).fill_(fill)
    return bool((seen == fill).all())


def within(got, want, bound, what=""):
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside their bound, worst "
        f"{float((d / bound).nan_to_num(nan=float('inf')).max()):.3g} times it")


def rel(got, want):
    return float(torch.linalg.norm(got.double() - want) / torch.linalg.norm(want))
