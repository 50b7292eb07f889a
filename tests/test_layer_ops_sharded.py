"""Rotary positions and 8-bit weights of the sharded decoder layer: which heads a rank turns and that its
positions go with its rows on two `gloo` ranks (the rotation itself in 64 bits on the CPU), and, on a GPU, the
shards of a layer one by one against the whole."""

from __future__ import annotations

import sys
import traceback
from pathlib import Path

import pytest
import torch

import layer_ops_ref as R
from test_tp_gloo import _cpu_linear, _init, _run

ROOT = Path(__file__).resolve().parents[1]


def _turn(q, k, positions, table, interleaved=False):
    for t in (q, k):
        t.copy_(R.rotate(t, positions, table, interleaved))


def _worker_positions(rank, world, port, errq):
    try:
        sys.path[:0] = [str(ROOT), str(ROOT / "tests")]
        import torch.distributed as dist

        from zcutlass_b200 import torch_ops
        from zcutlass_b200.tp import LayerShape, TPDecoderLinears, TPGroup

        _init(rank, world, port)
        torch_ops.rotary_ = _turn
        shape = LayerShape(hidden=32, intermediate=48, q_heads=4, kv_heads=2, head_dim=8)
        layer = TPDecoderLinears(shape, TPGroup.from_env(), "cpu", torch.float32, seed=5, chunks=2, linear_fn=_cpu_linear)
        table = torch_ops.rotary_table(50, 4)
        layer.enable_rotary(table, interleaved=True)
        g = torch.Generator().manual_seed(1)
        x, positions = torch.randn(6, 32, generator=g), torch.tensor([7, 0, 49, -1, 3, 3])
        out = layer.forward(x, positions=positions).clone()

        def gather(t, dim):
            parts = [None] * world
            dist.all_gather_object(parts, t)
            return torch.cat(parts, dim=dim)

        # q heads 0-3 and k heads 4, 5 of the whole output turned, v left as it is
        qkv = x @ gather(layer.qkv.weight, 0).t()
        qk = R.rotate(qkv[:, :48].view(6, 6, 8), positions, table, True).flatten(1)
        torch.testing.assert_close(gather(layer.buffers(6, "cpu", torch.float32)["qkv"], 1),
                                   torch.cat([qk.float(), qkv[:, 48:]], 1), rtol=1e-4, atol=1e-4)
        d_in = gather(layer.buffers(6, "cpu", torch.float32)["gate_up"][:, : layer.d_cols], 1)
        torch.testing.assert_close(out, d_in @ gather(layer.down.weight, 1).t(), rtol=1e-4, atol=1e-4)
        dist.barrier()
        dist.destroy_process_group()
    except Exception:
        errq.put((rank, traceback.format_exc()))
        raise


def test_positions_of_a_sharded_layer_world2_gloo():
    procs, msgs = _run(_worker_positions)
    assert not msgs, msgs
    assert all(p.exitcode == 0 for p in procs)


@pytest.mark.gpu
@pytest.mark.parametrize("world", [2, 4])
@pytest.mark.parametrize("tokens", [1, 70])
def test_shards_of_an_8_bit_layer_with_rotary(cuda_device, world, tokens):
    """Each rank's linears and heads in turn: column shards that are whole 128 x 128 blocks give the columns of the
    whole product, bit for bit, row shards its terms."""
    from zcutlass_b200 import torch_ops
    from zcutlass_b200.tp import LayerShape, TPDecoderLinears, TPGroup

    bf16 = torch.bfloat16
    shape = LayerShape(hidden=512, intermediate=1024, q_heads=8, kv_heads=4, head_dim=128)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(tokens, 512, generator=g, device="cuda").to(bf16)
    positions = torch.randint(0, 400, (tokens,), generator=g, device="cuda")
    table = torch_ops.rotary_table(400, 64, device="cuda")
    ranks = [TPDecoderLinears(shape, TPGroup(r, world), cuda_device, bf16, qkv_bias=True) for r in range(world)]
    whole = {name: torch.cat([getattr(r, name).weight for r in ranks], dim)
             for name, dim in (("qkv", 0), ("gate_up", 0), ("o_proj", 1), ("down", 1))}
    bias = torch.cat([r.qkv.bias for r in ranks])
    for r in ranks:
        r.quantize_fp8()
        r.enable_rotary(table)

    qkv = torch_ops.linear_fp8(x, *torch_ops.quantize_fp8(whole["qkv"], layout="blocks"), bias)
    q, k = torch_ops.rotary(qkv[:, :1024].unflatten(1, (8, 128)), qkv[:, 1024:1536].unflatten(1, (4, 128)), positions, table)
    want = torch.cat([q.flatten(1), k.flatten(1), qkv[:, 1536:]], 1)
    parts = []
    for r in ranks:
        out = torch.empty(tokens, r.qkv.weight.shape[0], device="cuda", dtype=bf16)
        r._check_positions(positions)
        r.qkv(x, out)
        r._rotate(out, positions)
        parts.append(out)
    assert torch.equal(torch.cat(parts, 1), want)

    for name, width in (("o_proj", shape.o_in), ("down", shape.intermediate)):
        xin = torch.randn(tokens, width, generator=g, device="cuda").to(bf16)
        terms, step = [], width // world
        for i, r in enumerate(ranks):
            xs = xin[:, i * step:(i + 1) * step]
            out = torch.empty(tokens, 512, device="cuda", dtype=bf16)
            getattr(r, name).partial(xs, out)
            w = getattr(r, name).weight
            R.check_product(out, *R.product(*R.quantize(xs, R.E4M3, 1), w.q, w.scale), step)
            terms.append((w.q, w.scale))
        q8, s8 = torch_ops.quantize_fp8(whole[name], layout="blocks")  # shards of whole blocks: the same values
        assert torch.equal(torch.cat([t[0].view(torch.uint8) for t in terms], 1), q8.view(torch.uint8))
        assert torch.equal(torch.cat([t[1] for t in terms], 1), s8)
