"""PyTorch operators backed by libzcutlass_torch.so.

Loading registers (CUDA dispatch key only):
    torch.ops.zcutlass_torch.gemm(A, B, C=None, bias=None, alpha=1.0, beta=0.0) -> D
    torch.ops.zcutlass.gemm(...)        same op, product namespace
    torch.ops.zcutlass.gemm_out(A, B, C, bias, alpha, beta, D) -> ()
    torch.ops.zcutlass.linear(x, weight[N, K], bias=None) -> y
    torch.ops.zcutlass.quantize_fp8(x, layout="rows", dtype=None) -> Tensor[]
    torch.ops.zcutlass.gemm_fp8(A, A_scale, B, B_scale, bias=None, out_dtype=None) -> D
    torch.ops.zcutlass.linear_fp8(x, weight, weight_scale, bias=None) -> y
    torch.ops.zcutlass.linear_fp8_out(x, weight, weight_scale, bias, out) -> ()
    torch.ops.zcutlass.linear_fp8_train(x, weight, bias=None) -> y   differentiable
    torch.ops.zcutlass.rotary(q, k, positions, table, interleaved=False, inverse=False) -> (q, k)
    torch.ops.zcutlass.rotary_(q, k, positions, table, ...) -> ()   in place

`selected_gemm_config` mirrors the reference's extension query
(python/zcutlass_torch/csrc/zcutlass_torch.cpp:91-149 in supercatking/zcutlass):
same checks, same dict keys, answered by the C ABI telemetry.
"""

from __future__ import annotations

import functools
import math
from pathlib import Path

from . import _native

TORCH_SO = Path(__file__).resolve().parent / "libzcutlass_torch.so"
_LOADED = False


def load() -> None:
    """Registers the torch operators; raises if the extension was not built."""
    global _LOADED
    if _LOADED:
        return
    import torch

    if not TORCH_SO.exists():
        raise ImportError(f"{TORCH_SO} is missing: build it with `python -m zcutlass_b200.build`")
    _native.lib()  # same process-wide copy of libzcutlass.so the operators link against
    torch.ops.load_library(str(TORCH_SO))
    _LOADED = True


def available() -> bool:
    try:
        load()
    except Exception:
        return False
    return True


def _dtype_code(t) -> int:
    import torch

    if t.dtype == torch.float16:
        return _native.F16
    if t.dtype == torch.bfloat16:
        return _native.BF16
    raise RuntimeError("zcutlass only supports float16 and bfloat16 tensors")


def _check_2d(t, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dim() != 2:
        raise RuntimeError(f"{name} must be rank-2")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be row-major contiguous")
    _dtype_code(t)


def selected_gemm_config(a, b, c=None, bias=None, alpha: float = 1.0, beta: float = 0.0) -> dict:
    """Dispatch metadata for one GEMM call site (host only, nothing launches)."""
    _check_2d(a, "A")
    _check_2d(b, "B")
    if a.dtype != b.dtype:
        raise RuntimeError("A and B dtype must match")
    if a.shape[1] != b.shape[0]:
        raise RuntimeError("A.shape[1] must equal B.shape[0]")
    if a.device != b.device:
        raise RuntimeError("A and B must be on the same CUDA device")
    if c is not None:
        _check_2d(c, "C")
        if c.dtype != a.dtype or c.device != a.device or tuple(c.shape) != (a.shape[0], b.shape[1]):
            raise RuntimeError("C must match A/B in dtype and device and be [A.shape[0], B.shape[1]]")
    if bias is not None:
        if not bias.is_cuda or bias.dim() != 1 or not bias.is_contiguous():
            raise RuntimeError("bias must be a contiguous rank-1 CUDA tensor")
        if bias.dtype != a.dtype or bias.shape[0] != b.shape[1]:
            raise RuntimeError("bias must match A/B dtype and have length B.shape[1]")
    t = _dtype_code(a)
    desc = _native.make_desc(a.shape[0], b.shape[1], a.shape[1], a.stride(0), b.stride(0),
                             c.stride(0) if c is not None else b.shape[1], b.shape[1], t,
                             float(alpha), float(beta), bias.data_ptr() if bias is not None else None)
    with _device_of(a):
        return _native.selected_kernel(desc)


class _device_of:
    """Makes `t.device` current so selection sees the right device's properties."""

    def __init__(self, t) -> None:
        self.t = t

    def __enter__(self):
        import torch

        self.ctx = torch.cuda.device(self.t.device)
        return self.ctx.__enter__()

    def __exit__(self, *exc):
        return self.ctx.__exit__(*exc)


def gemm(a, b, c=None, bias=None, alpha: float = 1.0, beta: float = 0.0):
    import torch

    load()
    return torch.ops.zcutlass.gemm(a, b, c, bias, float(alpha), float(beta))


def gemm_out(a, b, d, c=None, bias=None, alpha: float = 1.0, beta: float = 0.0):
    import torch

    load()
    torch.ops.zcutlass.gemm_out(a, b, c, bias, float(alpha), float(beta), d)
    return d


def linear(x, weight, bias=None):
    import torch

    load()
    return torch.ops.zcutlass.linear(x, weight, bias)


# ---------------------------------------------------------------- 8-bit linears


@functools.cache
def _op(name: str):
    """The registered operator (its only overload: a call on it skips the overload search)."""
    import torch

    load()
    return getattr(torch.ops.zcutlass, name).default


def quantize_fp8(x, layout: str = "rows", dtype=None) -> tuple:
    """x [R, C] (float16, bfloat16 or float32) in 8-bit floating point with a
    scale per group of 128: x ~= q * scale.

    layout  "rows"         (q [R, C], scale [R, ceil(C / 128)])
            "columns"      (q [C, R], scale [C, ceil(R / 128)]) of x.T: what a weight gradient reads
            "both"         the two of "rows", then the two of "columns", in one read of x
            "blocks"       (q [R, C], scale [ceil(R / 128), ceil(C / 128)]): weights
            "blocks_both"  the same, then the same values for x.T
    dtype   torch.float8_e4m3fn (default) or torch.float8_e5m2

    A scale is the smallest power of two (>= 2^-126) that keeps its group
    within the type's largest value, 1 for a group of zeros; q = x / scale
    rounded to nearest even. A group with an infinity or a NaN becomes NaN
    throughout, its scale too. Rows of q are padded to 16 bytes in memory
    (stride), as gemm_fp8 reads them fastest."""
    return tuple(_op("quantize_fp8")(x, layout, dtype))


def gemm_fp8(a, a_scale, b, b_scale, bias=None, out_dtype=None):
    """a [M, K] @ b [N, K].T (+ bias), both in 8-bit floating point (e4m3 or
    e5m2, mixed freely), accumulated in 32 bits and rounded once to out_dtype
    (bfloat16 by default, float16, float32).

    a_scale [M, ceil(K / 128)]; b_scale [N, ceil(K / 128)], or
    [ceil(N / 128), ceil(K / 128)] for weights in 128 x 128 blocks: float32 of
    any value and any strides (a product of two scales beyond 32 bits gives an
    infinity, NaN or 0). Rows whose stride is no multiple of 16 bytes, as
    .contiguous() leaves them where K is none, run without the tensor cores:
    about 100 times slower for large products."""
    return _op("gemm_fp8")(a, a_scale, b, b_scale, bias, out_dtype)


def linear_fp8(x, weight, weight_scale, bias=None):
    """x [..., K] @ weight [N, K].T (+ bias) with the weight held in 8 bits
    (quantize_fp8(w, "blocks"), or a checkpoint's values and scales) and x
    quantised by rows on the way in; y has x's dtype. For serving; training
    uses linear_fp8_train. Faster than the 16-bit linear for fewer than about
    128 rows of x and for more than 512, slower in between (251 x 8960 x 1536:
    13.3 us against 11.1; 512 x 4096 x 4096: 20.8 against 20.3)."""
    return _op("linear_fp8")(x, weight, weight_scale, bias)


def linear_fp8_out(x, weight, weight_scale, out, bias=None):
    """linear_fp8 of a matrix x [M, K] into out [M, N] (x's dtype, rows
    contiguous, any row stride); returns out."""
    _op("linear_fp8_out")(x, weight, weight_scale, bias, out)
    return out


def linear_fp8_train(x, weight, bias=None):
    """x [..., K] @ weight [N, K].T (+ bias) from unquantised operands, with
    all three products of a training step in 8-bit floating point (e4m3):

        y  = Q(x) Q(w).T + bias     x by rows, w in 128 x 128 blocks
        dx = Q(dy) Q(w)             dy by rows
        dw = Q(dy.T) Q(x.T).T       dy and x by columns
        db = sum of dy over tokens

    each accumulated in 32 bits and rounded once to x's dtype (dw: weight's).
    x, bias: one of float16, bfloat16, float32; weight: any of them. The
    backward pass keeps x and weight in 8 bits only. Capturing a step into a
    CUDA graph is refused while an eager graph of the same leaves is alive."""
    return _op("linear_fp8_train")(x, weight, bias)


# ---------------------------------------------------------------- rotary positions


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[list[float], float]:
    """(radians per position of each of the rotary_dim / 2 pairs, factor on
    cosines and sines). `scaling` stretches positions for long contexts:

        None                                  base^(-2 i / rotary_dim)
        {"type": "linear", "factor"}          all frequencies / factor
        {"type": "ntk", "factor"}             base * factor^(rotary_dim / (rotary_dim - 2))
        {"type": "llama3", "factor", "original", "low": 1, "high": 4}
            frequencies below `low` turns over the original length / factor,
            those above `high` turns kept, blended linearly in between
        {"type": "yarn", "factor", "original", "fast": 32, "slow": 1, "attention": 0.1 ln(factor) + 1}
            pair indices blended between those that turn `fast` and `slow`
            times over the original length; cosines and sines * attention"""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    half = rotary_dim // 2
    kind = "none" if scaling is None else scaling.get("type")
    if kind not in ("none", "linear", "ntk", "llama3", "yarn"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    factor = 1.0 if scaling is None else float(scaling["factor"])
    if not factor > 0 or not base > 0:
        raise ValueError("base and the scaling factor must be positive")
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(half)]
    if kind in ("none", "ntk"):
        return freq, 1.0
    if kind == "linear":
        return [f / factor for f in freq], 1.0
    original = float(scaling["original"])
    if not original > 0:
        raise ValueError("the original length must be positive")
    if kind == "llama3":
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if not high > low:
            raise ValueError("llama3 scaling needs high > low")
        keep = [min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low))) for f in freq]
        return [k * f + (1 - k) * f / factor for k, f in zip(keep, freq)], 1.0
    fast, slow = float(scaling.get("fast", 32.0)), float(scaling.get("slow", 1.0))

    def index(turns: float) -> float:  # the (real) pair index that makes `turns` turns over the original length
        return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
    span = max(hi - lo, 1e-3)
    keep = [1.0 - min(1.0, max(0.0, (i - lo) / span)) for i in range(half)]
    attention = float(scaling.get("attention", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
    return [k * f + (1 - k) * f / factor for k, f in zip(keep, freq)], attention


def rotary_table(positions: int, rotary_dim: int, base: float = 10000.0, scaling: dict | None = None, device=None):
    """[positions, rotary_dim] float32: the cosines of positions 0..positions-1
    in the first half of each row, the sines in the second. Angles and their
    functions are computed in 64 bits, so far positions stay exact. Made once
    and kept, for any number of layers and calls."""
    import torch

    freq, factor = rotary_frequencies(rotary_dim, base, scaling)
    if positions < 1:
        raise ValueError("positions must be at least 1")
    f = torch.tensor(freq, dtype=torch.float64, device=device)
    half = rotary_dim // 2
    table = torch.empty(positions, rotary_dim, dtype=torch.float32, device=device)
    for p0 in range(0, positions, 65536):  # bounds the 64-bit temporaries
        angle = torch.arange(p0, min(p0 + 65536, positions), dtype=torch.float64, device=device)[:, None] * f
        table[p0:p0 + 65536, :half] = angle.cos() * factor
        table[p0:p0 + 65536, half:] = angle.sin() * factor
    return table


def rotary(q, k, positions, table, interleaved: bool = False):
    """Rotary positions on q [tokens, q_heads, head_dim] and k [tokens,
    k_heads, head_dim] (float16, bfloat16 or float32, any token and head
    strides, so views of a packed qkv matrix serve); returns new tensors,
    differentiable in q and k.

    positions: int32 or int64 [tokens]; table: rotary_table(...), whose width
    is the rotary dimension (at most head_dim; the rest of a head is copied).
    interleaved: pairs (2 i, 2 i + 1) instead of (i, i + rotary_dim / 2).
    A negative position marks padding, whose heads are copied as they are. A
    position at or beyond the table's end does the same and sets the device
    error word (zcutlass_b200.tp.check_device_error raises on it)."""
    return _op("rotary")(q, k, positions, table, interleaved)


def rotary_(q, k, positions, table, interleaved: bool = False) -> None:
    """rotary() in place, without gradients."""
    import torch

    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        raise RuntimeError("rotary_ has no gradient: use rotary, or call it under torch.no_grad()")
    _op("rotary_")(q, k, positions, table, interleaved)
