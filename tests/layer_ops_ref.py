"""64-bit forms of the 8-bit quantiser, the block-scaled product and rotary positions, and error bounds."""

from __future__ import annotations

import torch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
MANTISSA = {E4M3: 3, E5M2: 2}
LEAST_EXPONENT = {E4M3: -6, E5M2: -14}


def groups(n: int) -> int:
    return -(-n // 128)


def two(k):
    """2^k in 64 bits (k: integer tensor), by the exponent's bits."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def quantize(x, dtype, block_rows: int):
    """(q, scale) in 64 bits of a matrix x: groups of block_rows x 128."""
    x = x.double()
    r, c = x.shape
    rb, cb = -(-r // block_rows), groups(c)
    grid = torch.zeros(rb * block_rows, cb * 128, dtype=torch.float64, device=x.device)
    grid[:r, :c] = x.abs()
    amax = grid.view(rb, block_rows, cb, 128).amax((1, 3))  # NaN propagates
    bad = ~torch.isfinite(amax)
    fit = torch.where(bad, 0.0, amax)
    k = torch.full_like(fit, -126).long()
    for step in (128, 64, 32, 16, 8, 4, 2, 1):  # the smallest k in [-126, 129] with amax <= largest * 2^k
        low = k + step - 1
        k = torch.where(fit > LARGEST[dtype] * two(low), k + step, k)
    s = torch.where(fit == 0, 1.0, two(k))
    s = torch.where(bad, torch.nan, s)
    each = s.repeat_interleave(block_rows, 0).repeat_interleave(128, 1)[:r, :c]
    t = x / each
    e = torch.frexp(t)[1] - 1
    spacing = two(torch.where(torch.isfinite(t), e, 0).clamp(min=LEAST_EXPONENT[dtype]) - MANTISSA[dtype])
    return torch.round(t / spacing) * spacing, s


def expand(scale, rows: int, cols: int):
    s = scale.double().repeat_interleave(128, 1)[:, :cols]
    return s if scale.shape[0] == rows else s.repeat_interleave(128, 0)[:rows]


def values(q, scale):
    return q.double() * expand(scale, *q.shape)


def product(a, a_scale, b, b_scale, bias=None):
    """(D, sum of absolute terms) in 64 bits."""
    va, vb = values(a, a_scale), values(b, b_scale)
    d, s = va @ vb.t(), va.abs() @ vb.abs().t()
    return (d, s) if bias is None else (d + bias.double(), s + bias.double().abs())


def half_ulp(ref, dtype):
    """Largest rounding error of a value near ref (|ref| may be off by the other errors: a relative bound
    of half an epsilon, and half the smallest subnormal)."""
    f = torch.finfo(dtype)
    return ref.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def check_product(d, ref, abs_sum, k: int):
    """|D - ref| <= one rounding to D's type + the roundings of a sum of k terms in 32 bits: at most one of
    2^-24 (relative to the sum of absolute values) per product, per block of 128 (scale product, scaling,
    addition) and for the bias."""
    steps = k + 3 * groups(k) + 2
    bound = abs_sum * (steps * 2.0 ** -24) * (1 + torch.finfo(d.dtype).eps) + half_ulp(ref, d.dtype)
    err = (d.double() - ref).abs()
    worst = (err / bound.clamp(min=1e-300)).max().item() if d.numel() else 0.0
    assert torch.isfinite(d).all()
    assert worst <= 1.0, f"error is {worst:.3g} of the bound"


def rotate(x, positions, table, interleaved, inverse=False):
    z = x.double().clone()
    r = table.shape[1]
    rows = table.double()[positions.clamp(0, max(table.shape[0] - 1, 0))]
    known = ((positions >= 0) & (positions < table.shape[0]))[:, None, None]
    c, s = rows[:, None, : r // 2], rows[:, None, r // 2:]
    s = -s if inverse else s
    i1 = torch.arange(0, r, 2, device=x.device) if interleaved else torch.arange(r // 2, device=x.device)
    i2 = i1 + 1 if interleaved else i1 + r // 2
    u, v = z[..., i1].clone(), z[..., i2].clone()
    z[..., i1] = torch.where(known, u * c - v * s, u)
    z[..., i2] = torch.where(known, v * c + u * s, v)
    return z


def check_rotated(y, x, positions, table, interleaved, inverse=False):
    """Two products and a sum in 32 bits (3 roundings of 2^-24 relative to |x1 c| + |x2 s| <= 2 |x|max of the
    pair times the table's largest entry), then one rounding to y's type."""
    ref = rotate(x, positions, table, interleaved, inverse)
    size = x.double().abs().amax(-1, keepdim=True) * 2 * max(1.0, table.abs().max().item()) if x.numel() else ref
    bound = half_ulp(ref, y.dtype) + size * (3 * 2.0 ** -24) * (1 + torch.finfo(y.dtype).eps)
    assert ((y.double() - ref).abs() <= bound).all()


# ---------------------------------------------------------------- gradients against differences


def aligned_signs(m: int, n: int, k: int, seed: int = 0):
    """x [m, k], w [n, k], c [m, n] in 32 bits, magnitudes in [0.5, 1.5], with signs s_m u_k, t_n u_k and
    s_m t_n: every term of y = x w^T, of c w and of c^T x has the sign of its sum, so nothing cancels."""
    g = torch.Generator().manual_seed(seed)
    s, t, u = (torch.randint(0, 2, (d,), generator=g) * 2.0 - 1.0 for d in (m, n, k))
    mag = lambda *d: torch.rand(*d, generator=g) + 0.5  # noqa: E731
    return s[:, None] * u * mag(m, k), t[:, None] * u * mag(n, k), s[:, None] * t * mag(m, n)


def difference_error(loss, x, other, c, grad, step: float = 4.0):
    """(error, bound): the derivative of loss(x) along v = sign(x), by a difference over x +- step v, against
    sum(grad * v), where loss(x) = sum(c * (Q(x) Q(other)^T)) and grad = Q(c) Q(other). A value a of a group
    with largest value A is off by at most 2^-4 (|a| + 2^-13 A) (half a step relative to the value, or half the
    smallest step), a product of two such by e = 2^-3 + 2^-8 of its absolute terms. With aligned_signs both
    errors are near e times the derivative itself: the bound is about a quarter of it."""
    v = torch.sign(x)
    diff = (loss(x + step * v) - loss(x - step * v)) / (2 * step)
    size = lambda t: t.double().abs() + 2.0 ** -13 * t.double().abs().max()  # noqa: E731
    e = 2.0 ** -3 + 2.0 ** -8 + 2.0 ** -16  # and the roundings of sums in 32 bits
    terms = (((size(x + step * v) + size(x - step * v)) @ size(other).t()) * c.double().abs()).sum() / (2 * step)
    grads = (size(c) @ size(other)).sum()
    return (diff - (grad.double() * v.double()).sum()).abs().item(), (e * (terms + grads)).item()
