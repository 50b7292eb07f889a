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
