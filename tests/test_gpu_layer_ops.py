"""GPU tests of the 8-bit linears (quantiser, block-scaled product, differentiable linear) and rotary
positions against 64-bit forms, through the public torch entry points."""

from __future__ import annotations

import pytest
import torch

import layer_ops_ref as R
from layer_ops_ref import E4M3, E5M2, groups
from zcutlass_b200 import torch_ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def same(got, want):
    """Bit-exact, NaN equal to NaN."""
    assert got.shape == want.shape
    assert torch.equal(torch.nan_to_num(got.double(), nan=12345.0), torch.nan_to_num(want.double(), nan=12345.0))


# ---------------------------------------------------------------- quantiser

SHAPES = [(1, 1), (1, 128), (3, 130), (8, 4096), (127, 257), (128, 128), (129, 1000), (300, 513), (1000, 48)]
LAYOUTS = ["rows", "columns", "both", "blocks", "blocks_both"]


def check_quantized(x, layout, dtype):
    out = torch_ops.quantize_fp8(x, layout=layout, dtype=dtype)
    block = 128 if layout.startswith("blocks") else 1
    want = []
    if layout != "columns":
        want += R.quantize(x, dtype, block)
    if layout in ("columns", "both", "blocks_both"):
        want += R.quantize(x.t(), dtype, block)
    assert len(out) == len(want)
    for i, (g, w) in enumerate(zip(out, want)):
        assert g.dtype == (dtype if i % 2 == 0 else F32)
        same(g, w)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("xt", [BF16, F16, F32], ids=str)
def test_quantize(cuda_device, shape, layout, xt):
    check_quantized(rand(*shape, seed=1, scale=3.0, dtype=xt), layout, E4M3)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_quantize_e5m2(cuda_device, layout):
    check_quantized(rand(200, 300, seed=2, scale=1e3), layout, E5M2)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("fp8", [E4M3, E5M2], ids=str)
def test_quantize_extremes(cuda_device, layout, fp8):
    """All exponents of 32-bit values, subnormals, zeros of both signs, exact borders, infinities and NaN."""
    x = torch.randint(0, 2 ** 31, (384, 512), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    x = (x.int() & 0x7f7fffff).view(F32).clone()  # finite, every exponent
    x[128:] *= 1e-30
    x[0:128, 128:256] = 0.0
    x[0:64, 128:256] *= -1.0
    x[256, 0:128] = 448.0 * 2.0 ** torch.randint(-100, 100, (128,), device="cuda")
    x[257, 0:128] = 2.0 ** -149
    x[258, 0] = float("inf")
    x[259, 200] = float("nan")
    x[260, 300] = -float("inf")
    check_quantized(x, layout, fp8)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("xt", [BF16, F32], ids=str)
def test_quantize_strided_and_unaligned(cuda_device, layout, xt):
    store = rand(130, 700, seed=4, dtype=xt)
    check_quantized(store[:, 3:603], layout, E4M3)     # unaligned rows
    check_quantized(store[::2, 8:520], layout, E4M3)   # every second row
    check_quantized(store[1:2, 1:2], layout, E4M3)


def test_quantize_empty(cuda_device):
    q, s = torch_ops.quantize_fp8(rand(0, 64))
    assert q.shape == (0, 64) and s.shape == (0, 1)
    q, s, qt, st = torch_ops.quantize_fp8(rand(64, 0), layout="both")
    assert q.shape == (64, 0) and s.shape == (64, 0) and qt.shape == (0, 64) and st.shape == (0, 1)


# ---------------------------------------------------------------- block-scaled product

GEMM_SHAPES = [(1, 1, 1), (1, 128, 128), (1, 300, 512), (5, 129, 1111), (16, 4096, 1024), (33, 256, 640), (64, 1000, 4096),
               (65, 64, 128), (100, 1, 200), (128, 128, 256), (200, 333, 777), (257, 511, 384), (300, 1024, 2048),
               (513, 1999, 1030), (1024, 1536, 512)]


def operands(m, n, k, b_rows, fa=E4M3, fb=E4M3, seed=0):
    a, sa = torch_ops.quantize_fp8(rand(m, k, seed=seed), dtype=fa)
    b, sb = torch_ops.quantize_fp8(rand(n, k, seed=seed + 1), layout="rows" if b_rows else "blocks", dtype=fb)
    sb = sb * (0.5 + torch.rand(sb.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
    return a, sa, b, sb


def check_gemm(a, sa, b, sb, out, bias=None):
    d = torch_ops.gemm_fp8(a, sa, b, sb, bias, out)
    assert d.dtype == out and d.is_contiguous()
    R.check_product(d, *R.product(a, sa, b, sb, bias), a.shape[1])
    return d


@pytest.mark.parametrize("b_rows", [False, True], ids=["b_blocks", "b_rows"])
@pytest.mark.parametrize("mnk", GEMM_SHAPES, ids=str)
@pytest.mark.parametrize("out", [BF16, F32], ids=str)
def test_gemm(cuda_device, mnk, b_rows, out):
    a, sa, b, sb = operands(*mnk, b_rows)
    check_gemm(a, sa, b, sb, out, rand(mnk[1], seed=9, dtype=out) if mnk[0] % 2 else None)


@pytest.mark.parametrize("fa,fb", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)], ids=str)
@pytest.mark.parametrize("mnk", [(7, 200, 300), (300, 520, 1000)], ids=str)
def test_gemm_types(cuda_device, mnk, fa, fb):
    a, sa, b, sb = operands(*mnk, True, fa, fb)
    check_gemm(a, sa, b, sb, F16)


KERNELS = ["fp8_generic", "fp8_tile16", "fp8_tile32", "fp8_tile64", "fp8_tile128", "fp8_pair"]


@pytest.mark.parametrize("b_rows", [False, True], ids=["b_blocks", "b_rows"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_gemm_every_kernel(cuda_device, monkeypatch, kernel, b_rows):
    """Each kernel over ragged edges in every dimension, odd and even counts of k blocks, several tiles per
    CTA, every output type, with and without bias, aligned and odd rows of D."""
    monkeypatch.setenv("ZCUTLASS_FORCE_KERNEL", kernel)
    for i, (m, n, k) in enumerate([(1, 1, 1), (16, 128, 128), (17, 200, 300), (130, 264, 1000), (300, 520, 384), (513, 777, 640),
                                   (256, 512, 1152)]):
        a, sa, b, sb = operands(m, n, k, b_rows, seed=i)
        for out in (BF16, F16, F32):
            check_gemm(a, sa, b, sb, out, rand(n, seed=9, dtype=out) if i % 2 else None)
    if kernel == "fp8_pair":  # more tiles than CTA pairs, an odd number of blocks
        a, sa, b, sb = operands(2500, 3000, 640, b_rows)
        check_gemm(a, sa, b, sb, BF16)


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("m", [3, 30, 60, 200])
def test_gemm_splits(cuda_device, monkeypatch, m, splits):
    monkeypatch.setenv("ZCUTLASS_SPLITK", str(splits))
    for n in (256, 333):
        a, sa, b, sb = operands(m, n, 2100, False)
        check_gemm(a, sa, b, sb, BF16, rand(n, seed=3, dtype=BF16))
        check_gemm(a, sa, b, sb, F32)


@pytest.mark.parametrize("m", [4, 40, 200, 600])
def test_gemm_strides(cuda_device, m):
    """Unpadded odd rows and offset bases (no TMA), scales in every stride order, views of larger buffers."""
    k, n = 333, 270
    a, sa, b, sb = operands(m, n, k, False)
    d = check_gemm(a, sa, b, sb, F32)
    pack = lambda t: t.view(torch.uint8).contiguous().view(t.dtype)  # noqa: E731
    for a2, b2 in ((pack(a), pack(b)), (a, pack(b)), (pack(a), b)):
        d2 = torch_ops.gemm_fp8(a2, sa.contiguous(), b2, sb.t().contiguous().t(), out_dtype=F32)
        R.check_product(d2, *R.product(a2, sa, b2, sb), k)
    wide = torch.zeros(m, 512, dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + k] = a.view(torch.uint8)
    spaced = torch.zeros(2 * m, 2 * groups(k), device="cuda")
    spaced[::2, ::2] = sa
    assert torch.equal(torch_ops.gemm_fp8(wide.view(E4M3)[:, 16:16 + k], spaced[::2, ::2], b, sb, out_dtype=F32), d)


def test_gemm_does_not_write_or_read_padding(cuda_device):
    """Poisoned bytes behind the rows of 8-bit operands do not reach the result."""
    m, n, k = 70, 150, 200
    a, sa, b, sb = operands(m, n, k, False)
    want = torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32)
    for t in (a, b):
        whole = t.view(torch.uint8).as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1))
        whole[:, k:] = 0x7f
    assert torch.equal(torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32), want)


@pytest.mark.parametrize("mnk", [(0, 64, 64), (64, 0, 64), (3, 200, 0), (300, 300, 0)], ids=str)
def test_gemm_empty(cuda_device, mnk):
    m, n, k = mnk
    a = torch.zeros(m, k, dtype=E4M3, device="cuda")
    b = torch.zeros(n, k, dtype=E4M3, device="cuda")
    bias = rand(n, dtype=BF16)
    d = torch_ops.gemm_fp8(a, torch.ones(m, groups(k), device="cuda"), b, torch.ones(groups(n), groups(k), device="cuda"), bias)
    assert torch.equal(d, bias.expand(m, n))


@pytest.mark.parametrize("m", [3, 300])
def test_gemm_nan_stays_in_its_row(cuda_device, m):
    x = rand(m, 512)
    x[1, 200] = float("nan")
    a, sa = torch_ops.quantize_fp8(x)
    b, sb = torch_ops.quantize_fp8(rand(256, 512, seed=1), layout="blocks")
    d = torch_ops.gemm_fp8(a, sa, b, sb)
    assert torch.isnan(d[1]).all() and torch.isfinite(d[0]).all() and torch.isfinite(d[2:]).all()


def test_gemm_same_bits_every_time(cuda_device):
    for mnk in ((16, 4096, 4096), (200, 1024, 4096), (1024, 2048, 1024)):
        a, sa, b, sb = operands(*mnk, False)
        d = torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32)
        for _ in range(5):
            assert torch.equal(torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32), d)


def check_linear(x, w, s, bias):
    y = torch_ops.linear_fp8(x, w, s, bias)
    x2 = x.reshape(-1, x.shape[-1])
    q, sx = R.quantize(x2, E4M3, 1)
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], w.shape[0])
    R.check_product(y.reshape(-1, w.shape[0]), *R.product(q, sx, w, s, bias), w.shape[1])


@pytest.mark.parametrize("xt", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("m", [1, 2, 16, 17, 47, 64, 129, 700])
def test_linear(cuda_device, m, xt):
    w, s = torch_ops.quantize_fp8(rand(768, 1000, seed=1, scale=0.03), layout="blocks")
    check_linear(rand(m, 1000, seed=2, dtype=xt), w, s, rand(768, seed=3, dtype=xt) if m % 2 else None)


def test_linear_shapes(cuda_device):
    w, s = torch_ops.quantize_fp8(rand(384, 256, seed=1, scale=0.05), layout="blocks")
    check_linear(rand(256, seed=2, dtype=BF16), w, s, None)
    check_linear(rand(2, 3, 5, 256, seed=2, dtype=BF16), w, s, None)
    check_linear(rand(256, 40, seed=2, dtype=BF16).t(), w, s, None)            # transposed input
    check_linear(rand(40, 600, seed=2, dtype=BF16)[:, 100:356], w, s, None)    # slice of a packed matrix
    check_linear(rand(1, 256, seed=2, dtype=BF16).expand(9, 256), w, s, None)  # one row for all
    assert torch_ops.linear_fp8(rand(0, 256, dtype=BF16), w, s).shape == (0, 384)


# ---------------------------------------------------------------- differentiable linear


@pytest.mark.parametrize("xt,wt", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32)], ids=str)
@pytest.mark.parametrize("mnk", [(1, 1, 1), (1, 130, 70), (130, 200, 333), (257, 384, 640), (1000, 520, 264)], ids=str)
def test_train(cuda_device, mnk, xt, wt):
    m, n, k = mnk
    x = rand(m, k, seed=1, dtype=xt).requires_grad_()
    w = rand(n, k, seed=2, scale=k ** -0.5, dtype=wt).requires_grad_()
    b = rand(n, seed=3, dtype=xt).requires_grad_()
    dy = rand(m, n, seed=4, dtype=xt)
    y = torch_ops.linear_fp8_train(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    qx, qw, qy = R.quantize(x.detach(), E4M3, 1), R.quantize(w.detach(), E4M3, 128), R.quantize(dy, E4M3, 1)
    R.check_product(y.detach(), *R.product(*qx, *qw, b.detach()), k)
    wt_q, wt_s = qw[0].t(), qw[1].t()
    R.check_product(dx, *R.product(*qy, wt_q, wt_s), n)
    R.check_product(dw, *R.product(*R.quantize(dy.t(), E4M3, 1), *R.quantize(x.detach().t(), E4M3, 1)), m)
    assert dx.dtype == xt and dw.dtype == wt and db.dtype == xt
    ref = dy.double().sum(0)
    bound = dy.double().abs().sum(0) * (m * 2.0 ** -24) + R.half_ulp(ref, xt) * (1 + 2.0 ** -8)
    assert ((db.double() - ref).abs() <= bound).all()


def test_train_only_what_is_asked(cuda_device):
    x, w, b = rand(64, 256, dtype=BF16), rand(128, 256, seed=1, dtype=BF16), rand(128, dtype=BF16)
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, True, False)):
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        torch_ops.linear_fp8_train(*leaves).sum().backward()  # an expanded gradient
        assert [t.grad is not None for t in leaves] == list(need)
    y = torch_ops.linear_fp8_train(x, w, b)
    assert not y.requires_grad


def test_train_leading_dimensions_and_no_tokens(cuda_device):
    w = rand(96, 160, seed=1, dtype=BF16).requires_grad_()
    x = rand(2, 7, 160, seed=2, dtype=BF16).requires_grad_()
    y = torch_ops.linear_fp8_train(x, w)
    y.backward(rand(2, 7, 96, seed=3, dtype=BF16))
    flat_x = x.detach().view(14, 160).requires_grad_()
    flat_w = w.detach().clone().requires_grad_()
    torch_ops.linear_fp8_train(flat_x, flat_w).backward(rand(2, 7, 96, seed=3, dtype=BF16).view(14, 96))
    assert torch.equal(x.grad.view(14, 160), flat_x.grad) and torch.equal(w.grad, flat_w.grad)
    b = rand(96, dtype=BF16).requires_grad_()
    x0, w0 = rand(0, 160, dtype=BF16).requires_grad_(), rand(96, 160, dtype=BF16).requires_grad_()
    torch_ops.linear_fp8_train(x0, w0, b).sum().backward()
    assert x0.grad.shape == (0, 160) and not w0.grad.any() and not b.grad.any()


def test_train_gradient_against_differences(cuda_device):
    """The loss is linear in the unquantised values up to quantisation: a difference over a step far above
    the quantisation step agrees with the gradient. A value v of a group with largest value a is off by at
    most 2^-4 |v|, or, below the normal range, half a step 2^-10 s <= 2^-17 a: together 2^-4 (|v| + 2^-13 a).
    A sum of products of two such factors is off by (2^-4 + 2^-4 + 2^-8) of its absolute terms."""
    m, n, k = 64, 96, 128
    x = rand(m, k, seed=1).requires_grad_()
    w = rand(n, k, seed=2).requires_grad_()
    c = rand(m, n, seed=3)
    torch_ops.linear_fp8_train(x, w).backward(c)
    v = rand(m, k, seed=4)
    plus = (torch_ops.linear_fp8_train(x.detach() + 4 * v, w.detach()).double() * c.double()).sum()
    minus = (torch_ops.linear_fp8_train(x.detach() - 4 * v, w.detach()).double() * c.double()).sum()
    size = lambda t: t.detach().double().abs() + 2.0 ** -13 * t.detach().double().abs().max()  # noqa: E731
    rel = 2.0 ** -3 + 2.0 ** -8
    terms = ((size(x) + 4 * size(v)) @ size(w).t() * size(c)).sum()
    grads = ((size(c) @ size(w)) * size(v)).sum()
    assert abs((plus - minus) / 8 - (x.grad.double() * v.double()).sum()) <= rel * (2 * terms / 8 + grads)


# ---------------------------------------------------------------- rotary positions


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (80, 80), (80, 20), (96, 48), (64, 2), (7, 6), (256, 256), (16, 0)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_rotary(cuda_device, dim, rot, dtype, interleaved):
    tokens, hq, hk = 37, 6, 2
    table = torch_ops.rotary_table(500, rot, device="cuda") if rot else torch.zeros(500, 0, device="cuda")
    q, k = rand(tokens, hq, dim, seed=1, dtype=dtype), rand(tokens, hk, dim, seed=2, dtype=dtype)
    pos = torch.randint(0, 500, (tokens,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    for p in (pos, pos.int()):
        qo, ko = torch_ops.rotary(q, k, p, table, interleaved)
        assert qo.is_contiguous() and ko.is_contiguous()
        if rot == 0:
            assert torch.equal(qo, q) and torch.equal(ko, k)
            continue
        R.check_rotated(qo, q, pos, table, interleaved)
        R.check_rotated(ko, k, pos, table, interleaved)


@pytest.mark.parametrize("tokens", [0, 1, 2, 1000, 5000])
@pytest.mark.parametrize("hq,hk", [(32, 8), (1, 1), (9, 0), (28, 4)], ids=str)
def test_rotary_sizes(cuda_device, tokens, hq, hk):
    table = torch_ops.rotary_table(4096, 128, device="cuda")
    q, k = rand(tokens, hq, 128, seed=1, dtype=BF16), rand(tokens, hk, 128, seed=2, dtype=BF16)
    pos = torch.arange(tokens, device="cuda") % 4096
    qo, ko = torch_ops.rotary(q, k, pos, table)
    R.check_rotated(qo, q, pos, table, False)
    R.check_rotated(ko, k, pos, table, False)


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_rotary_views_and_in_place(cuda_device, interleaved):
    tokens, hq, hk, d = 50, 8, 2, 64
    table = torch_ops.rotary_table(64, 32, device="cuda")
    pos = torch.arange(tokens, device="cuda")
    for offset in (0, 1):  # aligned, and off by one element
        store = rand(tokens, (hq + 2 * hk) * d + 8, seed=3, dtype=BF16)
        packed = store[:, offset:offset + (hq + 2 * hk) * d]
        q = packed[:, : hq * d].unflatten(1, (hq, d))
        k = packed[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
        before = store.clone()
        qo, ko = torch_ops.rotary(q, k, pos, table, interleaved)
        assert torch.equal(store, before)
        R.check_rotated(qo, q, pos, table, interleaved)
        torch_ops.rotary_(q, k, pos, table, interleaved)
        assert torch.equal(q, qo) and torch.equal(k, ko)
        touched = torch.zeros_like(store, dtype=torch.bool)
        touched[:, offset:offset + (hq + hk) * d] = True
        assert torch.equal(store[~touched], before[~touched])
    heads_first = rand(hq, tokens, d, seed=4, dtype=F16).transpose(0, 1)  # [heads, tokens, dim] storage
    qo, _ = torch_ops.rotary(heads_first, rand(tokens, hk, d, dtype=F16), pos, table, interleaved)
    R.check_rotated(qo, heads_first, pos, table, interleaved)


def test_rotary_padding_and_unknown_positions(cuda_device):
    from zcutlass_b200 import _native, tp

    table = torch_ops.rotary_table(16, 64, device="cuda")
    q, k = rand(4, 3, 64, seed=1), rand(4, 1, 64, seed=2)
    pos = torch.tensor([3, -1, 15, -(2 ** 40)], device="cuda")
    _native.device_error(clear=True)
    qo, ko = torch_ops.rotary(q, k, pos, table)
    assert torch.equal(qo[[1, 3]], q[[1, 3]]) and torch.equal(ko[[1, 3]], k[[1, 3]])
    R.check_rotated(qo, q, pos, table, False)
    tp.check_device_error()
    qo, _ = torch_ops.rotary(q, k, torch.tensor([3, 16, 15, 2 ** 40], device="cuda"), table)
    assert torch.equal(qo[[1, 3]], q[[1, 3]])
    with pytest.raises(RuntimeError, match="rotary position"):
        tp.check_device_error()
    tp.check_device_error()


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_rotary_gradient(cuda_device, dtype, interleaved):
    tokens = 33
    table = torch_ops.rotary_table(5000, 48, scaling={"type": "yarn", "factor": 4.0, "original": 1024}, device="cuda")
    pos = torch.randint(0, 5000, (tokens,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    q, k = rand(tokens, 4, 64, seed=1, dtype=dtype).requires_grad_(), rand(tokens, 2, 64, seed=2, dtype=dtype).requires_grad_()
    gq, gk = rand(tokens, 4, 64, seed=3, dtype=dtype), rand(tokens, 2, 64, seed=4, dtype=dtype)
    out = torch_ops.rotary(q, k, pos, table, interleaved)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk), retain_graph=True)
    R.check_rotated(dq, gq, pos, table, interleaved, inverse=True)
    R.check_rotated(dk, gk, pos, table, interleaved, inverse=True)
    (only_q,) = torch.autograd.grad(out[0].sum(), (q,))  # k unused, an expanded gradient
    R.check_rotated(only_q, torch.ones_like(gq), pos, table, interleaved, inverse=True)
    if dtype == F32:  # against a difference in the direction v: the map is linear
        v = rand(tokens, 4, 64, seed=5)
        with torch.no_grad():
            hi, _ = torch_ops.rotary(q + v, k, pos, table, interleaved)
            lo, _ = torch_ops.rotary(q - v, k, pos, table, interleaved)
        diff = ((hi.double() - lo.double()) * gq.double()).sum() / 2
        size = ((hi.double().abs() + lo.double().abs()) * gq.double().abs()).sum()
        assert abs(diff - (dq.double() * v.double()).sum()) <= 8 * 2.0 ** -24 * size


# ---------------------------------------------------------------- streams, graphs, refusals, together


def test_other_stream_and_graph(cuda_device):
    w, s = torch_ops.quantize_fp8(rand(512, 384, seed=1, scale=0.05), layout="blocks")
    table = torch_ops.rotary_table(100, 64, device="cuda")
    pos = torch.arange(48, device="cuda")
    x = rand(48, 384, seed=2, dtype=BF16)

    def step(x):
        y = torch_ops.linear_fp8(x, w, s)
        q, k = torch_ops.rotary(y[:, :256].unflatten(1, (4, 64)), y[:, 256:384].unflatten(1, (2, 64)), pos, table)
        return y, q, k

    want = [t.clone() for t in step(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, static = [], []
    for seed in (2, 3):  # two graphs alive at once, each with its own input
        xin = rand(48, 384, seed=seed, dtype=BF16)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(xin)
        graphs.append(g)
        static.append((xin, out))
    for xin, _ in static:
        xin.copy_(x)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out in static:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_backward_in_a_graph_beside_an_eager_graph(cuda_device):
    x, w = rand(64, 256, seed=1, dtype=BF16).requires_grad_(), rand(128, 256, seed=2, dtype=BF16).requires_grad_()
    table = torch_ops.rotary_table(64, 64, device="cuda")
    pos = torch.arange(64, device="cuda")
    dy = rand(64, 2, 64, seed=3, dtype=BF16)

    def step():
        y = torch_ops.linear_fp8_train(x, w).unflatten(1, (2, 64))
        q, _ = torch_ops.rotary(y, y[:, :1], pos, table)
        return torch.autograd.grad(q, (x, w), dy)

    want = [t.clone() for t in step()]
    y_eager = torch_ops.linear_fp8_train(x, w)  # an eager graph of the same leaves stays alive
    rotated = torch_ops.rotary(x.unflatten(1, (4, 64)), w.unflatten(1, (4, 64))[:64], pos, table)
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    y_eager.sum().backward()
    assert x.grad is not None and w.grad is not None
    del y_eager, rotated
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cuda_device):
    x = rand(64, 256, dtype=BF16)
    w, s = torch_ops.quantize_fp8(x, layout="blocks")
    a, sa = torch_ops.quantize_fp8(x)
    table = torch_ops.rotary_table(8, 64, device="cuda")
    q, pos = rand(8, 4, 64, dtype=BF16), torch.zeros(8, dtype=torch.long, device="cuda")
    bad = [
        lambda: torch_ops.quantize_fp8(x.double()),
        lambda: torch_ops.quantize_fp8(x[0]),
        lambda: torch_ops.quantize_fp8(x.t()),
        lambda: torch_ops.quantize_fp8(x[:1].expand(64, 256)),
        lambda: torch_ops.quantize_fp8(x, layout="diagonal"),
        lambda: torch_ops.quantize_fp8(x, dtype=BF16),
        lambda: torch_ops.quantize_fp8(x.clone().requires_grad_()),
        lambda: torch_ops.gemm_fp8(a, sa[:, :1], w, s),
        lambda: torch_ops.gemm_fp8(a, sa.half(), w, s),
        lambda: torch_ops.gemm_fp8(a, s, w, s),
        lambda: torch_ops.gemm_fp8(a[:, :128], sa[:, :1], w, s),
        lambda: torch_ops.gemm_fp8(x, sa, w, s),
        lambda: torch_ops.gemm_fp8(a, sa, w, s, out_dtype=torch.float64),
        lambda: torch_ops.gemm_fp8(a, sa, w, s, bias=rand(64, dtype=F32)),
        lambda: torch_ops.gemm_fp8(a, sa, w, s, bias=rand(63, dtype=BF16)),
        lambda: torch_ops.gemm_fp8(a.cpu(), sa, w, s),
        lambda: torch_ops.linear_fp8(x[:, :128], w, s),
        lambda: torch_ops.linear_fp8(x, x, s),
        lambda: torch_ops.linear_fp8(x.clone().requires_grad_(), w, s),
        lambda: torch_ops.linear_fp8_train(x, rand(8, 255, dtype=BF16)),
        lambda: torch_ops.linear_fp8_train(x, rand(8, 256, dtype=BF16), rand(8, dtype=F32)),
        lambda: torch_ops.rotary(q, q[:7], pos, table),
        lambda: torch_ops.rotary(q, q.half(), pos, table),
        lambda: torch_ops.rotary(q, q, pos[:7], table),
        lambda: torch_ops.rotary(q, q, pos.float(), table),
        lambda: torch_ops.rotary(q, q, pos, table.half()),
        lambda: torch_ops.rotary(q, q, pos, torch.zeros(8, 66, device="cuda")),
        lambda: torch_ops.rotary(q, q, pos, torch.zeros(8, 63, device="cuda")),
        lambda: torch_ops.rotary(q.transpose(1, 2), q.transpose(1, 2), pos, table),
        lambda: torch_ops.rotary_(q.clone().requires_grad_(), q, pos, table),
        lambda: torch_ops.rotary_(q, q, pos, table),
        lambda: torch_ops.rotary_(q, q[:, :1].expand(8, 4, 64), pos, table),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()


# ---------------------------------------------------------------- decoder layer


def layer_by_hand(layer, x, positions, table, interleaved):
    """The layer's chain, call by call."""
    s = layer.shape
    w = lambda linear: (linear.weight.q, linear.weight.scale)  # noqa: E731
    qkv = torch_ops.linear_fp8(x, *w(layer.qkv), layer.qkv.bias)
    q, k, _ = qkv.split([s.q_heads * s.head_dim, s.kv_heads * s.head_dim, s.kv_heads * s.head_dim], dim=1)
    q, k = torch_ops.rotary(q.unflatten(1, (-1, s.head_dim)), k.unflatten(1, (-1, s.head_dim)), positions, table, interleaved)
    o = torch_ops.linear_fp8(q.flatten(1), *w(layer.o_proj))
    gate_up = torch_ops.linear_fp8(o, *w(layer.gate_up))
    return torch_ops.linear_fp8(gate_up[:, : s.intermediate], *w(layer.down))


@pytest.mark.parametrize("tokens", [1, 24, 300])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_decoder_layer(cuda_device, tokens, interleaved):
    """8-bit linears and rotary positions in the tensor-parallel decoder layer: eagerly, over two streams
    and replayed from a graph, the same bits as the calls one by one."""
    from zcutlass_b200 import tp

    layer = tp.TPDecoderLinears(tp.LayerShape(512, 1280, 8, 2, 64), tp.TPGroup(), cuda_device, BF16, qkv_bias=True)
    x, positions = rand(tokens, 512, seed=1, dtype=BF16), torch.randint(0, 400, (tokens,), device="cuda")
    plain = layer.forward(x).clone()
    table = torch_ops.rotary_table(400, 48, device="cuda")
    layer.quantize_fp8()
    layer.quantize_fp8()
    eight = layer.forward(x).clone()
    assert not torch.equal(plain, eight)
    # four chained products of 8-bit factors: each factor off by at most 2^-4 of its value, errors of random
    # sign; the norm of the difference stays well below the norm of the result
    assert (eight.double() - plain.double()).norm() < 0.25 * plain.double().norm()
    layer.enable_rotary(table, interleaved)
    want = layer_by_hand(layer, x, positions, table, interleaved)
    assert torch.equal(layer.forward(x, positions=positions), want)
    if tokens > 1:
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        parts = [y.clone() for y in layer.forward_overlapped(x, streams, positions=positions)]
        torch.cuda.synchronize()
        h = tp.shard_range(tokens, 0, 2)[1]
        assert torch.equal(parts[0], layer_by_hand(layer, x[:h], positions[:h], table, interleaved))
        assert torch.equal(parts[1], layer_by_hand(layer, x[h:], positions[h:], table, interleaved))
    g = torch.cuda.CUDAGraph()
    xin, pin = x.clone(), positions.clone()
    with torch.cuda.graph(g):
        y = layer.forward(xin, positions=pin)
    xin.copy_(rand(tokens, 512, seed=7, dtype=BF16))
    pin.copy_(positions.flip(0))
    g.replay()
    assert torch.equal(y, layer_by_hand(layer, xin, pin, table, interleaved))


def test_linear_out(cuda_device):
    w, s = torch_ops.quantize_fp8(rand(300, 256, seed=1), layout="blocks")
    x, bias = rand(40, 256, seed=2, dtype=BF16), rand(300, seed=3, dtype=BF16)
    store = torch.full((40, 512), 7.0, device="cuda", dtype=BF16)
    for lo in (0, 3, 100):
        store.fill_(7.0)
        out = torch_ops.linear_fp8_out(x, w, s, store[:, lo:lo + 300], bias)
        assert torch.equal(out, torch_ops.linear_fp8(x, w, s, bias))
        assert (store[:, :lo] == 7.0).all() and (store[:, lo + 300:] == 7.0).all()
    for bad in (store, store[:, :300].float(), store[:39, :300]):
        with pytest.raises(RuntimeError):
            torch_ops.linear_fp8_out(x, w, s, bad, bias)


# ---------------------------------------------------------------- second derivatives, first calls, calls at once


def test_second_derivatives(cuda_device):
    table = torch_ops.rotary_table(32, 32, device="cuda")
    pos = torch.arange(9, device="cuda")
    q, k = rand(9, 2, 32, seed=1).requires_grad_(), rand(9, 1, 32, seed=2).requires_grad_()
    v = rand(9, 2, 32, seed=3).requires_grad_()
    out, _ = torch_ops.rotary(q, k, pos, table)
    (g,) = torch.autograd.grad(out, q, v, create_graph=True)
    u = rand(9, 2, 32, seed=4)
    (gg,) = torch.autograd.grad(g, v, u)  # the gradient is linear in v: its derivative turns u forward again
    R.check_rotated(gg, u, pos, table, False)
    x, w = rand(8, 64).requires_grad_(), rand(16, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(torch_ops.linear_fp8_train(x, w).sum(), x, create_graph=True)


def test_backward_computes_what_is_asked(cuda_device):
    """Gradients of one leaf alone, twice through one kept graph."""
    x, w = rand(40, 256, seed=1, dtype=BF16).requires_grad_(), rand(128, 256, seed=2, dtype=BF16).requires_grad_()
    dy = rand(40, 128, seed=3, dtype=BF16)
    y = torch_ops.linear_fp8_train(x, w)
    both = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, x, dy, retain_graph=True)[0], both[0])
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], both[1])


def test_first_calls_inside_a_capture(cuda_device):
    """A process whose first calls of every operator and kernel happen while a stream is captured."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from zcutlass_b200 import torch_ops as T
x = torch.randn(600, 1024, device="cuda").bfloat16()
big = torch.randn(2048, 1024, device="cuda")
table = T.rotary_table(600, 128, device="cuda")
pos = torch.arange(600, device="cuda")
torch.cuda.synchronize()
def step():
    w, s = T.quantize_fp8(big, layout="blocks")
    wr, sr = T.quantize_fp8(big, layout="rows")
    out = [T.linear_fp8(x[:m], w, s) for m in (1, 20, 50, 300, 600)]
    q, sq, _, _ = T.quantize_fp8(x, layout="both")
    out += [T.gemm_fp8(q[:m], sq[:m], wr, sr) for m in (1, 20, 50, 300, 600)]
    out += T.rotary(out[4][:, :1024].unflatten(1, (8, 128)), out[4][:, 1024:1280].unflatten(1, (2, 128)), pos, table)
    return out
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    captured = step()
g.replay()
torch.cuda.synchronize()
for a, b in zip(captured, step()):
    assert torch.equal(a, b)
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_calls_at_once_on_two_streams_and_threads(cuda_device):
    """Every kernel of the product beside itself and the others, from two threads."""
    import threading

    w, s = torch_ops.quantize_fp8(rand(1536, 2048, seed=1, scale=0.03), layout="blocks")
    xs = [rand(m, 2048, seed=m, dtype=BF16) for m in (1, 16, 30, 64, 200, 1500, 3000)]
    want = [torch_ops.linear_fp8(x, w, s) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(order):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = [(i, torch_ops.linear_fp8(xs[i], w, s)) for i in order]
            torch.cuda.current_stream().synchronize()
            wrong.extend(i for i, y in got if not torch.equal(y, want[i]))

    threads = [threading.Thread(target=work, args=(o,)) for o in (range(7), range(6, -1, -1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    from zcutlass_b200 import _native

    assert _native.device_error() == 0


@pytest.mark.parametrize("xt", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("m", [1, 3, 15, 16])
@pytest.mark.parametrize("k", [1, 100, 128, 130, 1000, 4096, 4200])
def test_linear_of_few_rows_has_the_bits_of_quantise_then_product(cuda_device, m, k, xt):
    """Odd widths, unaligned and strided rows, an infinity that stays in its row."""
    w, s = torch_ops.quantize_fp8(rand(390, k, seed=1, scale=k ** -0.5), layout="blocks")
    bias = rand(390, seed=2, dtype=xt)
    for x in (rand(m, k, seed=3, dtype=xt), rand(m, k + 9, seed=4, dtype=xt)[:, 3:3 + k], rand(2 * m, k + 8, seed=5, dtype=xt)[::2, :k]):
        q, sx = torch_ops.quantize_fp8(x.contiguous())
        want = torch_ops.gemm_fp8(q, sx, w, s, bias, xt)
        assert torch.equal(torch_ops.linear_fp8(x, w, s, bias), want)
    if m > 1:
        x = rand(m, k, seed=6, dtype=xt)
        x[1, k // 2] = float("inf")
        y = torch_ops.linear_fp8(x, w, s)
        assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 8])
def test_linear_of_few_rows_splits(cuda_device, monkeypatch, splits):
    monkeypatch.setenv("ZCUTLASS_SPLITK", str(splits))
    w, s = torch_ops.quantize_fp8(rand(256, 2500, seed=1, scale=0.02), layout="blocks")
    check_linear(rand(9, 2500, seed=2, dtype=BF16), w, s, None)


def test_linear_of_few_rows_with_unaligned_weights(cuda_device):
    w, s = torch_ops.quantize_fp8(rand(200, 333, seed=1, scale=0.05), layout="blocks")
    packed = w.view(torch.uint8).contiguous().view(E4M3)  # rows of 333 bytes: the generic kernel
    check_linear(rand(5, 333, seed=2, dtype=BF16), packed, s, None)
    w, s = torch_ops.quantize_fp8(rand(200, 256, seed=1, scale=0.05), layout="rows")  # a scale per row
    check_linear(rand(5, 256, seed=2, dtype=BF16), w, s, None)
