"""Host side of the 8-bit linears and rotary positions, without a GPU: argument checks of the C entry
points (they return before any CUDA work), rotary frequencies and tables, missing gradients."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import layer_ops_ref as R
from zcutlass_b200 import _native as N
from zcutlass_b200 import torch_ops

P = 0x1000  # aligned, non-null, never dereferenced


def quantize(x=P, q=P, scale=P, qt=None, scale_t=None, sums=None, **kw):
    base = dict(rows=64, cols=256, ldx=256, x_type=N.BF16, q_type=N.E4M3, block_rows=1, ldq=256, scale_row=1,
                scale_blk=64, ldqt=64, scale_t_row=1, scale_t_blk=256)
    base.update(kw)
    return N.lib().zcutlass_quantize_fp8(ctypes.byref(N.QuantizeDesc(**base)), x, q, scale, qt, scale_t, sums)


def gemm(a=P, sa=P, b=P, sb=P, d=P, **kw):
    base = dict(m=64, n=128, k=256, lda=256, ldb=256, ldd=128, a_type=N.E4M3, b_type=N.E4M3, d_type=N.BF16,
                b_scale_rows=128, a_scale_row=1, a_scale_blk=64, b_scale_row=2, b_scale_blk=1)
    base.update(kw)
    return N.lib().zcutlass_gemm_fp8(ctypes.byref(N.Fp8GemmDesc(**base)), a, sa, b, sb, d)


def rotary(q=P, qo=P, k=P, ko=P, pos=P, table=P, **kw):
    base = dict(tokens=4, q_heads=2, k_heads=1, head_dim=64, rotary_dim=64, dtype=N.BF16, positions64=1, q_token=128,
                q_head=64, q_out_token=128, q_out_head=64, k_token=64, k_head=64, k_out_token=64, k_out_head=64,
                table_rows=8, table_ld=64)
    base.update(kw)
    return N.lib().zcutlass_rotary(ctypes.byref(N.RotaryDesc(**base)), q, qo, k, ko, pos, table)


def test_quantize_arguments():
    bad, no = N.INVALID_ARGUMENT, N.NOT_SUPPORTED
    assert N.lib().zcutlass_quantize_fp8(None, P, P, P, None, None, None) == bad
    for kw in (dict(rows=-1), dict(cols=-1), dict(ldx=255), dict(ldq=255), dict(rows=2 ** 31), dict(x=None), dict(q=None),
               dict(scale=None), dict(qt=P), dict(qt=P, scale_t=P, ldqt=63), dict(sums=P), dict(x=P + 1), dict(scale=P + 2)):
        assert quantize(**kw) == bad, kw
    assert quantize(q=None, scale=None, qt=P, scale_t=P, sums=P, block_rows=128) == bad
    for kw in (dict(x_type=N.E4M3), dict(q_type=N.BF16), dict(q_type=N.E2M1), dict(block_rows=64)):
        assert quantize(**kw) == no, kw
    assert quantize(rows=0, x=None, q=None) == N.SUCCESS and quantize(cols=0) == N.SUCCESS
    assert N.lib().zcutlass_sum_rows(None, 4, 4, P, N.F32, None) == bad
    assert N.lib().zcutlass_sum_rows(P, 4, 4, P, N.E4M3, None) == no
    assert N.lib().zcutlass_sum_rows(None, 0, 0, None, N.F32, None) == N.SUCCESS


def test_gemm_arguments():
    bad, no = N.INVALID_ARGUMENT, N.NOT_SUPPORTED
    assert N.lib().zcutlass_gemm_fp8(None, P, P, P, P, P) == bad
    for kw in (dict(m=-1), dict(n=-1), dict(k=-1), dict(lda=255), dict(ldb=255), dict(ldd=127), dict(a=None), dict(sa=None),
               dict(b=None), dict(sb=None), dict(d=None), dict(k=2 ** 31, lda=2 ** 31, ldb=2 ** 31), dict(d=P + 1), dict(bias=P + 1),
               dict(sa=P + 2), dict(sb=P + 2), dict(d=P + 2, d_type=N.F32)):
        assert gemm(**kw) == bad, kw
    for kw in (dict(a_type=N.BF16), dict(b_type=N.F16), dict(d_type=N.E4M3), dict(a_type=N.E2M1), dict(b_scale_rows=64)):
        assert gemm(**kw) == no, kw
    assert gemm(m=0, a=None, d=None) == N.SUCCESS and gemm(n=0, b=None, d=None) == N.SUCCESS


def test_rotary_arguments():
    bad = N.INVALID_ARGUMENT
    assert N.lib().zcutlass_rotary(None, P, P, P, P, P, P) == bad
    for kw in (dict(tokens=-1), dict(q_heads=-1), dict(rotary_dim=63), dict(rotary_dim=66), dict(table_ld=63), dict(table_rows=-1),
               dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(pos=None), dict(table=None), dict(q=P + 1),
               dict(pos=P + 4), dict(table=P + 2), dict(head_dim=2 ** 20)):
        assert rotary(**kw) == bad, kw
    assert rotary(dtype=N.E4M3) == N.NOT_SUPPORTED
    assert rotary(tokens=0, q=None, pos=None) == N.SUCCESS
    assert rotary(q_heads=0, k_heads=0) == N.SUCCESS


# ---------------------------------------------------------------- frequencies and tables


def test_frequencies():
    f, a = torch_ops.rotary_frequencies(8, 10000.0)
    assert a == 1.0 and f == [1.0, 10000.0 ** -0.25, 10000.0 ** -0.5, 10000.0 ** -0.75]
    g, _ = torch_ops.rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert g == [x / 4 for x in f]
    g, _ = torch_ops.rotary_frequencies(8, 10000.0, {"type": "ntk", "factor": 4.0})
    assert g[0] == 1.0 and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-12)  # the lowest frequency is stretched by the factor
    g, _ = torch_ops.rotary_frequencies(128, 500000.0, {"type": "llama3", "factor": 8.0, "original": 8192})
    h, _ = torch_ops.rotary_frequencies(128, 500000.0)
    turns = [8192 * x / (2 * math.pi) for x in h]
    for t, x, y in zip(turns, g, h):
        assert x == y if t >= 4 else (x == y / 8 if t <= 1 else y / 8 < x < y)
    g, a = torch_ops.rotary_frequencies(128, 10000.0, {"type": "yarn", "factor": 16.0, "original": 4096})
    h, _ = torch_ops.rotary_frequencies(128, 10000.0)
    assert math.isclose(a, 0.1 * math.log(16.0) + 1) and g[0] == h[0] and math.isclose(g[-1], h[-1] / 16)
    ratio = [x / y for x, y in zip(g, h)]
    assert all(p >= q for p, q in zip(ratio, ratio[1:])) and any(1 / 16 < r < 1 for r in ratio)


def test_frequency_refusals():
    for args in ((7,), (0,), (-2,), (8, 0.0), (8, 1e4, {"type": "linear", "factor": 0.0}), (8, 1e4, {"type": "cubic", "factor": 2.0}),
                 (2, 1e4, {"type": "ntk", "factor": 2.0}), (8, 1e4, {"type": "yarn", "factor": 2.0, "original": 0}),
                 (8, 1e4, {"type": "llama3", "factor": 2.0, "original": 64, "low": 4, "high": 4})):
        with pytest.raises(ValueError):
            torch_ops.rotary_frequencies(*args)
    with pytest.raises(ValueError):
        torch_ops.rotary_table(0, 8)


def test_table_of_far_positions():
    n = 70000  # more than one chunk
    t = torch_ops.rotary_table(n, 6, base=100.0, scaling={"type": "yarn", "factor": 4.0, "original": 4096})
    assert t.shape == (n, 6) and t.dtype == torch.float32
    f, a = torch_ops.rotary_frequencies(6, 100.0, {"type": "yarn", "factor": 4.0, "original": 4096})
    for p in (0, 1, 65535, 65536, n - 1):
        for i in range(3):
            # one rounding to 32 bits (half a step), and 64-bit angles of up to 7e4 radians
            assert abs(t[p, i].item() - a * math.cos(p * f[i])) <= 2.0 ** -24 * a + 1e-10
            assert abs(t[p, 3 + i].item() - a * math.sin(p * f[i])) <= 2.0 ** -24 * a + 1e-10


def test_reference_quantiser():
    """The 64-bit form the GPU tests compare with, against hand-made values."""
    x = torch.tensor([[448.0, -1.0, 0.5, 2.0 ** -9, 3.0 * 2.0 ** -11]])
    q, s = R.quantize(x, R.E4M3, 1)
    assert s.item() == 1.0 and q.tolist() == [[448.0, -1.0, 0.5, 2.0 ** -9, 2.0 ** -9]]
    q, s = R.quantize(x * 1.001, R.E4M3, 1)
    assert s.item() == 2.0 and q[0, 0].item() == 224.0
    q, s = R.quantize(torch.zeros(2, 3), R.E5M2, 1)
    assert s.tolist() == [[1.0], [1.0]] and not q.any()
    q, s = R.quantize(torch.full((1, 2), 2.0 ** -149), R.E4M3, 128)
    assert s.item() == 2.0 ** -126 and not q.any()
    q, s = R.quantize(torch.tensor([[1.0, float("inf")]]), R.E4M3, 1)
    assert torch.isnan(s).all() and torch.isnan(q).all()


def test_no_gradient_is_refused():
    x = torch.zeros(4, 8, requires_grad=True)
    for call in (lambda: torch_ops.quantize_fp8(x), lambda: torch_ops.linear_fp8(x, x, x), lambda: torch_ops.gemm_fp8(x, x, x, x),
                 lambda: torch_ops.rotary_(x, x, None, None)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()


# ---------------------------------------------------------------- decoder layer


def test_no_gradient_of_tables_and_8_bit_operands_is_refused():
    """Operands without a gradient that require one: refused, not dropped from the graph."""
    torch_ops.load()
    q = torch.zeros(4, 2, 8)
    pos, table = torch.zeros(4, dtype=torch.int64), torch.zeros(16, 8)
    wq, s = torch.zeros(16, 128).to(torch.float8_e4m3fn), torch.ones(1, 1)
    x, xs = torch.zeros(4, 128), torch.ones(4, 1)
    grad_table, grad_w = table.clone().requires_grad_(), wq.clone().requires_grad_()
    a = torch.zeros(4, 128).to(torch.float8_e4m3fn)
    calls = [
        lambda: torch_ops.rotary(q, q, pos, grad_table),
        lambda: torch_ops.rotary(q.clone().requires_grad_(), q, pos, grad_table),
        lambda: torch_ops.rotary_(q, q, pos, grad_table),
        lambda: torch_ops.linear_fp8(x, grad_w, s),
        lambda: torch_ops.linear_fp8_out(x, grad_w, s, torch.zeros(4, 16)),
        lambda: torch_ops.gemm_fp8(a, xs, grad_w, s),
        lambda: torch_ops.gemm_fp8(a.clone().requires_grad_(), xs, wq, s),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()


def test_rotary_heads_of_a_shard():
    from zcutlass_b200 import tp

    s = tp.LLAMA3_8B  # 32 q, 8 k and 8 v heads of 128
    assert tp.rotary_heads(s, 0, s.qkv_out) == 40
    assert [tp.rotary_heads(s, *tp.shard_range(s.qkv_out, r, 4)) for r in range(4)] == [12, 12, 12, 4]
    assert sum(tp.rotary_heads(s, *tp.shard_range(s.qkv_out, r, 8)) for r in range(8)) == 40
    with pytest.raises(ValueError, match="whole heads"):
        tp.rotary_heads(s, 64, 1024)
    with pytest.raises(ValueError, match="whole heads"):
        tp.rotary_heads(tp.QWEN2_1_5B, *tp.shard_range(tp.QWEN2_1_5B.qkv_out, 0, 5))


def test_layer_positions_go_with_rotary():
    from zcutlass_b200 import tp

    def linear(x, w, bias, out):
        out.copy_(x @ w.t())

    layer = tp.TPDecoderLinears(tp.LayerShape(64, 128, 4, 2, 16), tp.TPGroup(), "cpu", torch.float32, linear_fn=linear)
    x = torch.randn(5, 64)
    y = layer.forward(x).clone()
    with pytest.raises(ValueError, match="positions"):
        layer.forward(x, positions=torch.arange(5))
    with pytest.raises(ValueError, match="wider"):
        layer.enable_rotary(torch.zeros(8, 32))
    assert torch.equal(layer.forward(x), y)
    layer.enable_rotary(torch_ops.rotary_table(8, 16))
    with pytest.raises(ValueError, match="positions"):
        layer.forward(x)
