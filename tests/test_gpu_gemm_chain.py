"""Products whose C and bias are what the kernel before on the stream has just written."""

from __future__ import annotations

import pytest
import torch

from zcutlass_b200 import torch_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mnk", [(256, 256, 256), (512, 4096, 512), (2048, 4096, 320), (4096, 4096, 256)], ids=str)
def test_chain_through_c_and_bias(cuda_device, mnk):
    """D = A B + C + bias with the C and the bias of the product before, without and with a wait in between."""
    m, n, k = mnk
    torch_ops.load()
    g = torch.Generator(device="cuda").manual_seed(1)
    a = [(torch.randn(m, k, generator=g, device="cuda") * k ** -0.5).bfloat16() for _ in (0, 1)]
    b = torch.randn(k, n, generator=g, device="cuda").bfloat16()

    def chain(wait):
        d = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
        for i in range(12):
            d = torch.ops.zcutlass.gemm(a[i % 2], b, d, d[i], 1.0, 0.5)
            if wait:
                torch.cuda.synchronize()
        return d

    want = chain(True)
    assert torch.isfinite(want).all()
    for _ in range(10):
        assert torch.equal(chain(False), want)
