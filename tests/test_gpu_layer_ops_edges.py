"""GPU tests of the 8-bit linears and rotary positions where kernels meet: column groups beyond the last
column of a split product, operands that the kernel before on the stream has just written, buffers handed
back between the CTAs of a pair."""

from __future__ import annotations

import pytest
import torch

import layer_ops_ref as R
from zcutlass_b200 import _native, torch_ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rand(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("splits", [2, 5, 8])
@pytest.mark.parametrize("n", [1, 4, 100, 129, 300])
def test_split_product_with_groups_beyond_the_last_column(cuda_device, monkeypatch, n, splits):
    """Clusters in which some CTAs own no column of D, launched back to back."""
    monkeypatch.setenv("ZCUTLASS_SPLITK", str(splits))
    for m in (1, 20, 64, 200):
        a, sa = torch_ops.quantize_fp8(rand(m, 2100, seed=m))
        b, sb = torch_ops.quantize_fp8(rand(n, 2100, seed=n), layout="blocks")
        d = [torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32) for _ in range(30)]
        R.check_product(d[0], *R.product(a, sa, b, sb), 2100)
        assert all(torch.equal(x, d[0]) for x in d)
    assert _native.device_error() == 0


@pytest.mark.parametrize("layout", ["blocks", "rows"])
@pytest.mark.parametrize("m", [1, 40, 200, 2400])
def test_scales_that_the_kernel_before_has_just_written(cuda_device, m, layout):
    """Two inputs in turn through recycled buffers, nothing waited for in between."""
    w = [rand(1100, 1500, seed=s) * 2.0 ** (5 * s) for s in (0, 1)]
    x = [rand(m, 1500, seed=s + 2) * 2.0 ** (7 * s) for s in (0, 1)]

    def step(i):
        b, sb = torch_ops.quantize_fp8(w[i], layout=layout)
        a, sa = torch_ops.quantize_fp8(x[i])
        return torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32)

    want = []
    for i in (0, 1):
        want.append(step(i))
        torch.cuda.synchronize()
    wrong = torch.zeros((), device="cuda", dtype=torch.int64)
    for t in range(40):
        wrong += (step(t % 2) != want[t % 2]).sum()
    assert wrong.item() == 0


@pytest.mark.parametrize("rot", [64, 6])
def test_rotary_table_that_the_kernel_before_has_just_written(cuda_device, rot):
    q, k = rand(500, 4, 64, seed=1), rand(500, 2, 64, seed=2)
    pos = torch.arange(500, device="cuda") % 300
    b, sb = torch_ops.quantize_fp8(rand(rot, 256, seed=3), layout="rows")
    a = [torch_ops.quantize_fp8(rand(300, 256, seed=4 + i)) for i in (0, 1)]

    def step(i):
        table = torch_ops.gemm_fp8(*a[i], b, sb, out_dtype=F32)
        return torch_ops.rotary(q, k, pos, table)

    want = []
    for i in (0, 1):
        want.append(step(i))
        torch.cuda.synchronize()
        R.check_rotated(want[i][0], q, pos, torch_ops.gemm_fp8(*a[i], b, sb, out_dtype=F32), False)
    wrong = torch.zeros((), device="cuda", dtype=torch.int64)
    for t in range(100):
        got = step(t % 2)
        wrong += sum((x != y).sum() for x, y in zip(got, want[t % 2]))
    assert wrong.item() == 0


@pytest.mark.parametrize("layout", ["blocks", "rows"])
def test_pair_product_hands_buffers_and_scales_back(cuda_device, monkeypatch, layout):
    """Many k blocks, each with scales far from its neighbours' (a block scaled by another's is off by 2^5 or
    more), several tiles per pair, beside memory traffic on another stream."""
    monkeypatch.setenv("ZCUTLASS_FORCE_KERNEL", "fp8_pair")
    m, n, k = 2300, 2500, 4224
    swing = (2.0 ** (5 * (torch.arange(33, device="cuda") % 7))).repeat_interleave(128)
    a, sa = torch_ops.quantize_fp8(rand(m, k, seed=1) * swing)
    b, sb = torch_ops.quantize_fp8(rand(n, k, seed=2) / swing, layout=layout)
    want = torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32)
    R.check_product(want, *R.product(a, sa, b, sb), k)
    torch.cuda.synchronize()
    noise = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    wrong = torch.zeros((), device="cuda", dtype=torch.int64)
    for _ in range(20):
        with torch.cuda.stream(side):
            noise.add_(1)
        wrong += (torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32) != want).sum()
    torch.cuda.synchronize()
    assert wrong.item() == 0 and _native.device_error() == 0


def test_rotary_refuses_more_heads_than_it_counts(cuda_device):
    """Sizes past 32 bits are refused before the result is allocated, not cut to their low bits."""
    table, pos = torch.zeros(4, 2, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    one = rand(1, 1, 2, dtype=BF16)
    for q, k in ((one.expand(1, 2 ** 32 + 2, 2), one), (one, one.expand(1, 2 ** 32 + 2, 2)),
                 (one.expand(1, 65537, 2), one), (rand(1, 1, 1).expand(1, 1, 65538), rand(1, 1, 1).expand(1, 1, 65538))):
        before = torch.cuda.memory_allocated()
        with pytest.raises(RuntimeError, match="at most 65536|contiguous heads"):
            torch_ops.rotary(q, k, pos, table)
        assert torch.cuda.memory_allocated() == before


def test_position_beyond_the_table_is_not_an_expired_wait(cuda_device):
    """It is reported, but apart: a wait that expires later still reports its own code, and kernels that skip
    their work once a wait has expired do not take the position for one."""
    table = torch_ops.rotary_table(16, 64, device="cuda")
    q = rand(4, 3, 64, seed=1)
    _native.device_error(clear=True)
    torch_ops.rotary(q, q, torch.tensor([3, 16, 15, 1], device="cuda"), table)
    assert _native.lib().zcutlass_selftest_bounded_wait(2000) == (15 << 4) | 15
    assert _native.device_error(clear=False) == (32 << 4) | 1
    assert _native.device_error(clear=True) == (32 << 4) | 1
    assert _native.device_error() == 0


@pytest.mark.parametrize("mnk", [(64, 96, 128), (130, 200, 260), (300, 512, 640)], ids=str)
def test_train_gradients_agree_with_differences(cuda_device, mnk):
    """Of x and of w, in directions in which no term cancels (layer_ops_ref.difference_error: what the bound
    tells apart is tested on the CPU)."""
    x, w, c = (t.cuda() for t in R.aligned_signs(*mnk, seed=2))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    torch_ops.linear_fp8_train(xg, wg).backward(c)
    of_x = lambda v: (torch_ops.linear_fp8_train(v, w).double() * c.double()).sum()  # noqa: E731
    of_w = lambda v: (torch_ops.linear_fp8_train(x, v).double() * c.double()).sum()  # noqa: E731
    for loss, leaf, other, grad, cc in ((of_x, x, w, xg.grad, c), (of_w, w, x, wg.grad, c.t())):
        error, bound = R.difference_error(loss, leaf, other, cc, grad)
        assert error <= bound
        for wrong in (grad * 0, -grad, grad.roll(1, 0), grad.roll(1, 1)):
            error, bound = R.difference_error(loss, leaf, other, cc, wrong)
            assert error > bound


def test_capture_is_refused_where_an_eager_graph_of_an_upstream_leaf_lives(cuda_device):
    """Views of a leaf, and what was computed from it, are refused as the leaf itself is."""
    qkv = rand(32, 8 * 64, seed=1, dtype=BF16).requires_grad_()
    w = rand(128, 512, seed=2, dtype=BF16).requires_grad_()
    table, pos = torch_ops.rotary_table(32, 64, device="cuda"), torch.arange(32, device="cuda")
    dy = rand(32, 6, 64, seed=3, dtype=BF16)

    def turn():
        q, _ = torch_ops.rotary(qkv[:, :384].unflatten(1, (6, 64)), qkv[:, 384:].unflatten(1, (2, 64)), pos, table)
        return torch.autograd.grad(q, qkv, dy)

    def project():
        return torch_ops.linear_fp8_train(qkv * 2, w)

    want = turn()[0].clone()
    eager = qkv * 3  # any graph of the leaf
    for step in (turn, project):
        with pytest.raises(RuntimeError, match="before capturing"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                step()
    del eager
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = turn()[0]
    g.replay()
    assert torch.equal(got, want)


def test_two_streams_of_one_capture_share_a_leaf(cuda_device):
    w = rand(128, 256, seed=1, dtype=BF16).requires_grad_()
    x = [rand(40, 256, seed=2 + i, dtype=BF16) for i in (0, 1)]
    dy = rand(40, 128, seed=4, dtype=BF16)
    side = torch.cuda.Stream()

    def step():
        here = torch.cuda.current_stream()
        y0 = torch_ops.linear_fp8_train(x[0], w)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            y1 = torch_ops.linear_fp8_train(x[1], w)
        here.wait_stream(side)
        return (y0.detach(), y1.detach()) + torch.autograd.grad((y0, y1), w, (dy, dy))

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("k", [300, 768, 896, 1280, 1536, 1792, 2560])
@pytest.mark.parametrize("m", [1, 16, 20, 64])
def test_short_products_of_few_rows(cuda_device, m, k):
    """K of few blocks: every count of splits that the choice can come to, over few and many tiles."""
    for n in (1, 256, 1000, 2048, 4096):
        a, sa = torch_ops.quantize_fp8(rand(m, k, seed=m))
        b, sb = torch_ops.quantize_fp8(rand(n, k, seed=n), layout="blocks")
        R.check_product(torch_ops.gemm_fp8(a, sa, b, sb, out_dtype=F32), *R.product(a, sa, b, sb), k)
