"""What the 8-bit linears and the rotary positions of zcutlass_b200 are measured on.

Four operators, each in a plain form (elementary torch operations in 32 bits, rounded once) and, where
`own` is true, as a user calls them in `zcutlass_b200.torch_ops`:

  quantize  x -> (q, s): 8-bit floating-point values with one power-of-two scale for 1 x 128 values of a
            row, of a column (the transposed operand of a weight gradient), both in one pass, or for
            128 x 128 blocks (weights). s = 2^ceil(log2(amax / max)), q = x / s rounded to nearest even.
  linear    y = x @ w^T + bias with w held in 8 bits (128 x 128 scales) and x quantised on the way in.
  gemm      D[m, n] = sum_b sa[m, b] * sb[n, b] * sum_{k in b} a[m, k] * b[n, k] on operands held in 8 bits.
  train     the linear from unquantised weights, forward and backward, all three products in 8 bits.
  rotary    rotary positions on q and k heads, half or interleaved pairs, whole heads or part of them,
            forward alone or with the gradients.

Inputs are synthetic: activations with a few outlier channels and some all-zero (padding) rows, weights
of variance 1 / in_features. Layer sizes are those of the layer shapes in zcutlass_b200.tp.
"""

from __future__ import annotations

import math

import torch

own = False

GROUP = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
# largest finite value of each 8-bit type, 1.75 * 2^TOP
TOP = {"e4m3": 8, "e5m2": 15}


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one decode step's activations before a projection: launch latency
        {"name": "quantize rows 8x4096", "op": "quantize", "rows": 8, "cols": 4096, "dtype": "bf16", "layout": "rows", "fp8": "e4m3"},
        # a training step's activations, quantised along both axes in one read
        {"name": "quantize both 8192x4096", "op": "quantize", "rows": 8192, "cols": 4096, "dtype": "bf16", "layout": "both", "fp8": "e4m3"},
        # 32-bit master weights of an MLP, requantised after an optimiser step
        {"name": "quantize blocks 14336x4096", "op": "quantize", "rows": 14336, "cols": 4096, "dtype": "f32", "layout": "blocks", "fp8": "e4m3"},
        # qkv projection of one decoded token
        {"name": "linear 1x6144x4096", "op": "linear", "m": 1, "n": 6144, "k": 4096, "dtype": "bf16", "bias": False},
        # down projection of a decode batch that fills no tile
        {"name": "linear 48x4096x14336", "op": "linear", "m": 48, "n": 4096, "k": 14336, "dtype": "bf16", "bias": False},
        # a short ragged prompt through a small model's gate projection, 16-bit floats with bias
        {"name": "linear 251x8960x1536", "op": "linear", "m": 251, "n": 8960, "k": 1536, "dtype": "f16", "bias": True},
        # gate and up projections of a long prefill, the largest product of the layer
        {"name": "linear 8192x28672x4096", "op": "linear", "m": 8192, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        # a weight-gradient product on its own: odd sizes, scales per row on both sides, 32-bit result
        {"name": "gemm 1111x1999x2035", "op": "gemm", "m": 1111, "n": 1999, "k": 2035, "fp8a": "e5m2", "fp8b": "e4m3", "b_rows": True, "out": "f32"},
        # forward and backward of one MLP projection in training
        {"name": "train 4096x14336x4096", "op": "train", "m": 4096, "n": 14336, "k": 4096, "dtype": "bf16", "bias": True},
        # one decode step's q and k heads
        {"name": "rotary decode 16", "op": "rotary", "tokens": 16, "q_heads": 32, "k_heads": 8, "head_dim": 128, "rotary_dim": 128, "interleaved": False,
         "dtype": "bf16", "packed": True, "grad": False, "far": 8192, "scaled": False},
        # a long prefill, read from the packed qkv output
        {"name": "rotary prefill 8192", "op": "rotary", "tokens": 8192, "q_heads": 32, "k_heads": 8, "head_dim": 128, "rotary_dim": 128, "interleaved": False,
         "dtype": "bf16", "packed": True, "grad": False, "far": 131072, "scaled": True},
        # training: interleaved pairs in half of each head, forward and gradients
        {"name": "rotary train 4001 part", "op": "rotary", "tokens": 4001, "q_heads": 12, "k_heads": 2, "head_dim": 128, "rotary_dim": 64, "interleaved": True,
         "dtype": "f16", "packed": False, "grad": True, "far": 32768, "scaled": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "gemm", "train", "rotary"])
    if op == "quantize":
        rows, cols = _log(rng, 1, 16384), _log(rng, 64, 14336)
        layout = rng.choice(["rows", "columns", "both", "blocks"])
        return {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(["bf16", "f16", "f32"]), "layout": layout, "fp8": rng.choice(["e4m3", "e4m3", "e5m2"])}
    if op == "linear":
        m = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 64, 8192)
        return {"op": op, "m": m, "n": _log(rng, 256, 28672), "k": _log(rng, 256, 4096 if m > 1024 else 14336),
                "dtype": rng.choice(["bf16", "f16"]), "bias": rng.random() < 0.5}
    if op == "gemm":
        return {"op": op, "m": _log(rng, 1, 6000), "n": _log(rng, 64, 8192), "k": _log(rng, 64, 8192), "fp8a": rng.choice(["e4m3", "e5m2"]),
                "fp8b": "e4m3", "b_rows": rng.random() < 0.5, "out": rng.choice(["bf16", "f16", "f32"])}
    if op == "train":
        return {"op": op, "m": _log(rng, 64, 4096), "n": _log(rng, 256, 8192), "k": _log(rng, 256, 4096), "dtype": rng.choice(["bf16", "f16"]),
                "bias": rng.random() < 0.5}
    head_dim = rng.choice([64, 80, 96, 112, 128, 256])
    k_heads = rng.choice([1, 2, 4, 8])
    return {"op": op, "tokens": _log(rng, 1, 8192), "q_heads": k_heads * rng.choice([1, 4, 6, 8]) if k_heads < 8 else rng.choice([8, 32]), "k_heads": k_heads,
            "head_dim": head_dim, "rotary_dim": rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4]), "interleaved": rng.random() < 0.4,
            "dtype": rng.choice(["bf16", "f16", "f32"]), "packed": rng.random() < 0.5, "grad": rng.random() < 0.5,
            "far": rng.choice([4096, 32768, 131072]), "scaled": rng.random() < 0.3}


# ---------------------------------------------------------------- inputs


def _activations(gen, rows, cols, dtype):
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.01, 20.0, 1.0)  # outlier channels
    if rows > 8:
        x *= (torch.rand(rows, 1, generator=gen, device="cuda") >= 0.01).float()  # padding tokens
    return x.to(dtype)


def _padded(q):
    """q in rows whose stride is a multiple of 16 bytes, as the framework keeps 8-bit operands."""
    rows, cols = q.shape
    store = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=q.device).view(q.dtype)
    store[:, :cols] = q
    return store[:, :cols]


def _far_table(case, device):
    """[far, rotary_dim] in 32 bits, cosines before sines; angles in 64 bits. `scaled`: the low frequencies
    stretched by 8 beyond an original length of 8192, blended between 1 and 4 turns."""
    r = case["rotary_dim"]
    freq = torch.pow(torch.tensor(500000.0 if case["scaled"] else 10000.0, dtype=torch.float64), -torch.arange(0, r, 2, dtype=torch.float64) / r)
    if case["scaled"]:
        turns = 8192 * freq / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        freq = keep * freq + (1 - keep) * freq / 8
    angle = torch.arange(case["far"], dtype=torch.float64, device=device)[:, None] * freq.to(device)[None, :]
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "quantize":
        s["x"] = _activations(gen, case["rows"], case["cols"], DTYPES[case["dtype"]])
    elif op == "linear":
        m, n, k, dtype = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        s["x"] = _activations(gen, m, k, dtype)
        q, s["w_scale"] = _quantize_blocks(torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5, "e4m3")
        s["w"] = _padded(q)
        s["bias"] = torch.randn(n, generator=gen, device="cuda").to(dtype) if case["bias"] else None
    elif op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        q, s["a_scale"] = _quantize_rows(_activations(gen, m, k, torch.float32), case["fp8a"])
        s["a"] = _padded(q)
        b = torch.randn(n, k, generator=gen, device="cuda")
        q, s["b_scale"] = _quantize_rows(b, case["fp8b"]) if case["b_rows"] else _quantize_blocks(b, case["fp8b"])
        s["b"] = _padded(q)
        # scales of checkpoints are no powers of two
        s["b_scale"] = s["b_scale"] * (0.5 + torch.rand(s["b_scale"].shape, generator=gen, device="cuda"))
    elif op == "train":
        m, n, k, dtype = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        s["x"] = _activations(gen, m, k, dtype).requires_grad_()
        s["w"] = (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).to(dtype).requires_grad_()
        s["bias"] = torch.randn(n, generator=gen, device="cuda").to(dtype).requires_grad_() if case["bias"] else None
        s["dy"] = (_activations(gen, m, n, torch.float32) * 2.0 ** -6).to(dtype)
    else:
        t, hq, hk, d, dtype = case["tokens"], case["q_heads"], case["k_heads"], case["head_dim"], DTYPES[case["dtype"]]
        if case["packed"]:  # views of a packed [tokens, q | k | v] projection
            qkv = torch.randn(t, (hq + 2 * hk) * d, generator=gen, device="cuda").to(dtype)
            s["q"] = qkv[:, : hq * d].view(t, hq, d)
            s["k"] = qkv[:, hq * d: (hq + hk) * d].view(t, hk, d)
        else:
            s["q"] = torch.randn(t, hq, d, generator=gen, device="cuda").to(dtype)
            s["k"] = torch.randn(t, hk, d, generator=gen, device="cuda").to(dtype)
        s["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device="cuda")
        s["table"] = _far_table(case, "cuda")
        if case["grad"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            s["dq"] = torch.randn(t, hq, d, generator=gen, device="cuda").to(dtype)
            s["dk"] = torch.randn(t, hk, d, generator=gen, device="cuda").to(dtype)
    return s


# ---------------------------------------------------------------- plain forms


def _power(amax, fp8):
    """The smallest power of two s with amax <= max * s (1 where all is zero, no less than 2^-126)."""
    f, e = torch.frexp(amax)
    k = (torch.where(f <= 0.875, e - 1, e) - TOP[fp8]).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), k), 1.0)


def _quantize_rows(x, fp8):
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    xp = torch.nn.functional.pad(x.float(), (0, groups * GROUP - cols)).view(rows, groups, GROUP)
    s = _power(xp.abs().amax(2), fp8)
    q = (xp / s[:, :, None]).to(FP8[fp8]).view(rows, groups * GROUP)[:, :cols]
    return q, s


def _quantize_blocks(x, fp8):
    rows, cols = x.shape
    rb, cb = -(-rows // GROUP), -(-cols // GROUP)
    xp = torch.nn.functional.pad(x.float(), (0, cb * GROUP - cols, 0, rb * GROUP - rows)).view(rb, GROUP, cb, GROUP)
    s = _power(xp.abs().amax((1, 3)), fp8)
    q = (xp / s[:, None, :, None]).to(FP8[fp8]).view(rb * GROUP, cb * GROUP)[:rows, :cols]
    return q, s


def _values(q, s):
    """The 32-bit values that q and its scales stand for."""
    rows, cols = q.shape
    s = s.repeat_interleave(GROUP, 1)[:, :cols]
    if s.shape[0] != rows:
        s = s.repeat_interleave(GROUP, 0)[:rows]
    return q.float() * s


def _plain_linear(x, w, bias):
    y = x @ w.t()
    return y if bias is None else y + bias.float()


def _turn(x, table, case, back):
    """x1 cos - x2 sin, x2 cos + x1 sin on the rotary part of each head (sines negated for the gradient)."""
    r = case["rotary_dim"]
    cos, sin = table[:, None, : r // 2], table[:, None, r // 2:]
    sin = -sin if back else sin
    f = x.float()
    if case["interleaved"]:
        a, b = f[..., 0:r:2], f[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = f[..., : r // 2], f[..., r // 2: r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, f[..., r:]], -1).to(x.dtype)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from zcutlass_b200 import torch_ops

        if op == "quantize":
            return torch_ops.quantize_fp8(state["x"], layout=case["layout"], dtype=FP8[case["fp8"]])
        if op == "linear":
            return torch_ops.linear_fp8(state["x"], state["w"], state["w_scale"], state["bias"])
        if op == "gemm":
            return torch_ops.gemm_fp8(state["a"], state["a_scale"], state["b"], state["b_scale"], out_dtype=DTYPES[case["out"]])
        if op == "train":
            y = torch_ops.linear_fp8_train(state["x"], state["w"], state["bias"])
            leaves = [state["x"], state["w"]] + ([] if state["bias"] is None else [state["bias"]])
            return (y.detach(),) + torch.autograd.grad(y, leaves, state["dy"])
        q, k = torch_ops.rotary(state["q"], state["k"], state["positions"], state["table"], interleaved=case["interleaved"])
        if not case["grad"]:
            return q, k
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))

    with torch.no_grad():
        if op == "quantize":
            x, fp8, layout = state["x"], case["fp8"], case["layout"]
            if layout == "blocks":
                return _quantize_blocks(x, fp8)
            along = _quantize_rows(x, fp8) if layout != "columns" else ()
            across = _quantize_rows(x.t(), fp8) if layout != "rows" else ()
            return tuple(along) + tuple(across)
        if op == "linear":
            y = _plain_linear(_values(*_quantize_rows(state["x"], "e4m3")), _values(state["w"], state["w_scale"]), state["bias"])
            return y.to(state["x"].dtype)
        if op == "gemm":
            return (_values(state["a"], state["a_scale"]) @ _values(state["b"], state["b_scale"]).t()).to(DTYPES[case["out"]])
        if op == "train":
            x, w, dy, dtype = state["x"], state["w"], state["dy"], state["x"].dtype
            wv = _values(*_quantize_blocks(w, "e4m3"))
            y = _plain_linear(_values(*_quantize_rows(x, "e4m3")), wv, state["bias"])
            dx = _values(*_quantize_rows(dy, "e4m3")) @ wv
            dw = _values(*_quantize_rows(dy.t(), "e4m3")) @ _values(*_quantize_rows(x.t(), "e4m3")).t()
            out = (y.to(dtype), dx.to(dtype), dw.to(dtype))
            return out if state["bias"] is None else out + (dy.float().sum(0).to(dtype),)
        table = state["table"][state["positions"]]
        out = (_turn(state["q"], table, case, False), _turn(state["k"], table, case, False))
        return out if not case["grad"] else out + (_turn(state["dq"], table, case, True), _turn(state["dk"], table, case, True))


# ---------------------------------------------------------------- 64 bits


def _two(k):
    """2^k in 64 bits, exactly, by the exponent's own bits."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _exact_quantize(x, fp8, block_rows):
    """(q, s, values) of x in 64 bits: groups of block_rows x 128, q on the type's grid by its spacing."""
    x = x.double()
    rows, cols = x.shape
    top, bits, least = (448.0, 3, -6) if fp8 == "e4m3" else (57344.0, 2, -14)
    grid = torch.zeros(-(-rows // block_rows) * block_rows, -(-cols // 128) * 128, dtype=torch.float64, device=x.device)
    grid[:rows, :cols] = x.abs()
    amax = grid.unfold(0, block_rows, block_rows).unfold(1, 128, 128).amax((2, 3))
    k = torch.floor(torch.log2(amax.clamp(min=1e-300) / top)) - 1  # too small; raised until amax fits
    for _ in range(3):
        k = torch.where(amax > top * _two(k), k + 1, k)
    s = _two(k.clamp(min=-126.0))
    s[amax == 0] = 1.0
    each = s.repeat_interleave(block_rows, 0).repeat_interleave(128, 1)[:rows, :cols]
    t = x / each
    spacing = _two(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** least))) - bits)
    q = torch.round(t / spacing) * spacing
    return q, s, q * each


def _exact_values(q, s):
    rows, cols = q.shape
    r = torch.arange(rows, device=q.device) // (1 if s.shape[0] == rows else 128)
    c = torch.arange(cols, device=q.device) // 128
    return q.double() * s.double()[r][:, c]


def _exact_turn(x, angles_cos, angles_sin, r, interleaved, sign):
    z = x.double().clone()
    first = torch.arange(0, r, 2, device=x.device) if interleaved else torch.arange(0, r // 2, device=x.device)
    second = first + 1 if interleaved else first + r // 2
    u, v = z[..., first], z[..., second]
    c, s = angles_cos.double()[:, None], sign * angles_sin.double()[:, None]
    z[..., first] = u * c - v * s
    z[..., second] = u * s + v * c
    return z


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "quantize":
            out = ()
            if case["layout"] == "blocks":
                return _exact_quantize(state["x"], case["fp8"], 128)[:2]
            if case["layout"] != "columns":
                out += _exact_quantize(state["x"], case["fp8"], 1)[:2]
            if case["layout"] != "rows":
                out += _exact_quantize(state["x"].t(), case["fp8"], 1)[:2]
            return out
        if op == "linear":
            y = torch.mm(_exact_quantize(state["x"], "e4m3", 1)[2], _exact_values(state["w"], state["w_scale"]).t())
            return y if state["bias"] is None else y + state["bias"].double()
        if op == "gemm":
            return torch.mm(_exact_values(state["a"], state["a_scale"]), _exact_values(state["b"], state["b_scale"]).t())
        if op == "train":
            x, w, dy = state["x"].detach(), state["w"].detach(), state["dy"]
            w8 = _exact_quantize(w, "e4m3", 128)[2]
            y = torch.mm(_exact_quantize(x, "e4m3", 1)[2], w8.t())
            dx = torch.mm(_exact_quantize(dy, "e4m3", 1)[2], w8)
            dw = torch.mm(_exact_quantize(dy.t(), "e4m3", 1)[2], _exact_quantize(x.t(), "e4m3", 1)[2].t())
            if state["bias"] is None:
                return y, dx, dw
            return y + state["bias"].detach().double(), dx, dw, dy.double().sum(0)
        r, inter = case["rotary_dim"], case["interleaved"]
        rows = state["table"][state["positions"]]
        cos, sin = rows[:, : r // 2], rows[:, r // 2:]
        out = tuple(_exact_turn(state[n].detach(), cos, sin, r, inter, 1.0) for n in ("q", "k"))
        if case["grad"]:
            out += tuple(_exact_turn(state[n], cos, sin, r, inter, -1.0) for n in ("dq", "dk"))
        return out


# ---------------------------------------------------------------- work


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    up = lambda v: -(-v // GROUP)  # noqa: E731
    op = case["op"]
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        n, ways = rows * cols, 2 if case["layout"] == "both" else 1
        scales = {"rows": rows * up(cols), "columns": cols * up(rows), "both": rows * up(cols) + cols * up(rows), "blocks": up(rows) * up(cols)}[case["layout"]]
        return {"bytes": n * size[case["dtype"]] + ways * n + 4 * scales, "flops": 2 * n}
    if op == "linear":
        m, n, k, e = case["m"], case["n"], case["k"], size[case["dtype"]]
        return {"bytes": m * k * e + n * k + 4 * up(n) * up(k) + m * n * e + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k + 4 * (m + (n if case["b_rows"] else up(n))) * up(k) + m * n * size[case["out"]], "flops": 2 * m * n * k}
    if op == "train":
        m, n, k, e = case["m"], case["n"], case["k"], size[case["dtype"]]
        # x, w and dy in; y, dx and dw out
        return {"bytes": 2 * (m * k + n * k + m * n) * e + (2 * n * e if case["bias"] else 0), "flops": 6 * m * n * k}
    t, r = case["tokens"], case["rotary_dim"]
    values = t * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
    turned = t * (case["q_heads"] + case["k_heads"]) * r
    ways = 2 if case["grad"] else 1
    return {"bytes": ways * 2 * values * size[case["dtype"]] + t * (8 + 4 * r), "flops": ways * 3 * turned}
