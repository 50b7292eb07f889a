"""Host side of the 8-bit linears and rotary positions, without a GPU: calls that would lose something
without a word are refused, and refusals say what they refuse."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import layer_ops_ref as R
from zcutlass_b200 import torch_ops

E4M3 = torch.float8_e4m3fn


def operands():
    torch_ops.load()
    return dict(x=torch.ones(4, 128), w=torch.ones(16, 128), bias=torch.ones(16), s=torch.ones(1, 1), xs=torch.ones(4, 1),
                q=torch.ones(4, 2, 8), pos=torch.zeros(4, dtype=torch.int64), table=torch.zeros(16, 8), out=torch.ones(4, 16))


# (operator, operand that carries the derivative, call)
CALLS = [
    ("quantize_fp8", "x", lambda o: torch_ops.quantize_fp8(o["x"])),
    ("gemm_fp8", "xs", lambda o: torch_ops.gemm_fp8(o["x"].detach().to(E4M3), o["xs"], o["w"].to(E4M3), o["s"])),
    ("gemm_fp8", "s", lambda o: torch_ops.gemm_fp8(o["x"].to(E4M3), o["xs"], o["w"].to(E4M3), o["s"])),
    ("linear_fp8", "x", lambda o: torch_ops.linear_fp8(o["x"], o["w"].to(E4M3), o["s"])),
    ("linear_fp8", "bias", lambda o: torch_ops.linear_fp8(o["x"], o["w"].to(E4M3), o["s"], o["bias"])),
    ("linear_fp8_out", "x", lambda o: torch_ops.linear_fp8_out(o["x"], o["w"].to(E4M3), o["s"], o["out"])),
    ("linear_fp8_out", "out", lambda o: torch_ops.linear_fp8_out(o["x"], o["w"].to(E4M3), o["s"], o["out"])),
    ("linear_fp8_train", "x", lambda o: torch_ops.linear_fp8_train(o["x"], o["w"])),
    ("linear_fp8_train", "w", lambda o: torch_ops.linear_fp8_train(o["x"], o["w"], o["bias"])),
    ("linear_fp8_train", "bias", lambda o: torch_ops.linear_fp8_train(o["x"], o["w"], o["bias"])),
    ("rotary", "q", lambda o: torch_ops.rotary(o["q"], o["q"].detach() * 1, o["pos"], o["table"])),
    ("rotary", "table", lambda o: torch_ops.rotary(o["q"], o["q"], o["pos"], o["table"])),
    ("rotary_", "q", lambda o: torch_ops.rotary_(o["q"], torch.ones(4, 2, 8), o["pos"], o["table"])),
]


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
@pytest.mark.parametrize("name,operand,call", CALLS, ids=lambda v: v if isinstance(v, str) else "")
def test_forward_mode_is_refused(name, operand, call, grad):
    """A tangent is refused, not dropped: in dual numbers and in torch.func.jvp, with and without no_grad (which
    does not switch forward mode off)."""
    o = operands()
    t = o[operand]
    match = f"{name} has no forward-mode derivative"
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        o[operand] = forward_ad.make_dual(t, torch.ones_like(t))
        with pytest.raises(RuntimeError, match=match):
            call(o)
    if grad:
        with pytest.raises(RuntimeError, match=match):
            torch.func.jvp(lambda v: call({**operands(), operand: v}), (t,), (torch.ones_like(t),))
    o[operand] = t  # without a tangent, the call goes on to its own checks
    with pytest.raises(RuntimeError, match="CUDA|cuda"):
        call(o)


def test_rotary_on_cpu_tensors_says_so():
    o = operands()
    for call in (torch_ops.rotary, torch_ops.rotary_):
        with pytest.raises(RuntimeError, match="q must be a rank-3 CUDA tensor"):
            call(o["q"], o["q"].clone(), o["pos"], o["table"])


def test_layer_with_its_own_linear_refuses_8_bit_weights():
    """Its function takes tensors; it must not be handed anything else."""
    from zcutlass_b200 import tp

    def linear(x, w, bias, out):
        out.copy_(x @ w.t())

    layer = tp.TPDecoderLinears(tp.LayerShape(64, 128, 4, 2, 16), tp.TPGroup(), "cpu", torch.float32, linear_fn=linear)
    x = torch.randn(5, 64)
    y = layer.forward(x).clone()
    with pytest.raises(ValueError, match="linear_fn"):
        layer.quantize_fp8()
    assert torch.equal(layer.forward(x), y)  # nothing was replaced


def test_difference_bound_tells_wrong_gradients():
    """The bound that the GPU test of the differentiable linear uses holds for the formulas in 64 bits, and no
    mistake passes it: no gradient, the wrong sign, rows or columns in another order, half of the sum."""
    x, w, c = R.aligned_signs(64, 96, 128, seed=1)
    product = lambda a, b: R.values(*R.quantize(a, E4M3, 1)) @ R.values(*b).t()  # noqa: E731
    blocks = lambda t: R.quantize(t, E4M3, 128)  # noqa: E731
    along = lambda t: R.quantize(t, E4M3, 1)  # noqa: E731
    turned = lambda q: (q[0].t(), q[1].t())  # noqa: E731
    dx, dw = product(c, turned(blocks(w))), product(c.t(), along(x.t()))
    of_x = lambda v: (product(v, blocks(w)) * c.double()).sum()  # noqa: E731
    of_w = lambda v: (product(x, blocks(v)) * c.double()).sum()  # noqa: E731
    for loss, leaf, other, grad, cc in ((of_x, x, w, dx, c), (of_w, w, x, dw, c.t())):
        error, bound = R.difference_error(loss, leaf, other, cc, grad)
        assert error <= bound
        for wrong in (grad * 0, -grad, grad.roll(1, 0), grad.roll(1, 1), grad * 0.5):
            error, bound = R.difference_error(loss, leaf, other, cc, wrong)
            assert error > bound


def test_rotary_head_limit_is_an_error_not_a_crash():
    """On tensors of CUDA's type without storage: the check comes before any work."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    torch_ops.load()
    with FakeTensorMode():
        one = torch.empty(1, 1, 2, device="cuda")
        pos, table = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.empty(4, 2, device="cuda")
        for heads in (65537, 2 ** 32 + 2):
            for q, k in ((one.expand(1, heads, 2), one), (one, one.expand(1, heads, 2))):
                with pytest.raises(RuntimeError, match="at most 65536"):
                    torch_ops.rotary(q, k, pos, table)
