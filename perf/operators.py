"""The feed-forward half of a transformer block on packed tokens, as measurable cases: the residual add with its
root-mean-square norm (result in 16 / 32 bits, or in 8 bits with scales), the matrix product of 8-bit operands with a scale per
block of 128, and the gated projections act(x Wg^T) * (x Wu^T) in 8 bits and, with their gradients, in 16 bits.

``run`` computes the plain form (elementary torch operations in float32) where ``own`` is false and makes the calls of a user
of this package where it is true.  An 8-bit result is a float8_e4m3fn tensor beside its scales.

Sizes: width 1024 with a hidden width of 4096 * 2 / 3 rounded up to a multiple of 8 (2736) is the gated form of the blocks of
``come_b200/vggt_arch.py``; 1374 tokens are one unmerged frame, 6456 and 80,672 the packed rows of the 8-frame and the
100-frame scene, 10,534 one GPU's share of the latter.
"""
from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
SMALLEST = E4M3_MAX * 2.0 ** -126  # block maxima below this take its scale, so that a scale is a normal number
BLOCK = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a single token between two products (a camera token refined on its own): launch latency
        {"name": "norm8 1x1024", "op": "norm", "dtype": "bf16", "tokens": 1, "width": 1024, "eight": True},
        # every MLP of the 100-frame scene
        {"name": "norm8 80672x1024", "op": "norm", "dtype": "bf16", "tokens": 80672, "width": 1024, "eight": True},
        # a float32 stream of a width that no block of 128 divides
        {"name": "norm 10534x1000 f32", "op": "norm", "dtype": "f32", "tokens": 10534, "width": 1000, "eight": False},
        # the down projection of a single token
        {"name": "linear8 1x2736-1024", "op": "linear8", "dtype": "bf16", "tokens": 1, "width": 2736, "out": 1024, "bias": True},
        # the attention's output projection, one unmerged frame
        {"name": "linear8 1374x1024-1024", "op": "linear8", "dtype": "f16", "tokens": 1374, "width": 1024, "out": 1024, "bias": True},
        # the down projection of the 100-frame scene
        {"name": "linear8 80672x2736-1024", "op": "linear8", "dtype": "bf16", "tokens": 80672, "width": 2736, "out": 1024, "bias": False},
        # the gated projections in 8 bits: a single token, the 8-frame and the 100-frame scene
        {"name": "gated8 1x1024-2736", "op": "gated8", "dtype": "e4m3", "tokens": 1, "width": 1024, "out": 2736, "bias": False, "act": "silu"},
        {"name": "gated8 6456x1024-2736", "op": "gated8", "dtype": "e4m3", "tokens": 6456, "width": 1024, "out": 2736, "bias": True, "act": "silu"},
        {"name": "gated8 80672x1024-2736", "op": "gated8", "dtype": "e4m3", "tokens": 80672, "width": 1024, "out": 2736, "bias": False, "act": "silu"},
        # a single token in 16 bits, inference
        {"name": "gated 1x1024-2736", "op": "gated", "dtype": "bf16", "tokens": 1, "width": 1024, "out": 2736, "bias": False, "act": "silu", "train": False},
        # a training step of a small head: odd numbers of tokens and of hidden channels, biases, the other activation
        {"name": "gated step 1001x392-1003", "op": "gated", "dtype": "f16", "tokens": 1001, "width": 392, "out": 1003, "bias": True, "act": "gelu", "train": True},
        # a training step on the tokens of an 8-frame scene
        {"name": "gated step 6456x1024-2736", "op": "gated", "dtype": "bf16", "tokens": 6456, "width": 1024, "out": 2736, "bias": False, "act": "silu", "train": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "linear8", "gated8", "gated"))
    if op == "norm":
        return {"op": op, "dtype": rng.choice(("f32", "f16", "bf16")), "tokens": _log_int(rng, 1, 60000), "width": 8 * _log_int(rng, 8, 160),
                "eight": rng.random() < 0.6}
    # 8-bit rows are stored with a stride of whole 16 bytes, so their width may be anything; 16-bit rows need widths of whole 16 bytes
    case = {"op": op, "tokens": _log_int(rng, 1, 40000), "width": 8 * _log_int(rng, 8, 250) if op == "gated" else _log_int(rng, 64, 2800),
            "out": _log_int(rng, 40, 2800), "bias": rng.random() < 0.5}
    if op == "linear8":
        return {**case, "dtype": rng.choice(("f32", "f16", "bf16"))}
    case["act"] = rng.choice(("silu", "gelu"))
    if op == "gated8":
        return {**case, "dtype": rng.choice(("e4m3", "e4m3", "f16", "bf16"))}
    case["train"] = rng.random() < 0.6
    if case["train"]:  # no drawn step costs more than the largest listed one
        case["tokens"] = min(case["tokens"], 6456)
        case["width"], case["out"] = min(case["width"], 1024), min(case["out"], 2736)
    return {**case, "dtype": rng.choice(("f16", "bf16"))}


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _random(seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=gen, device="cuda")


def _tokens(randn, tokens, width):
    """Rows as a residual stream has them: of unlike size, a few channels much larger than the rest."""
    channel = torch.exp(0.5 * randn(width))
    channel[:: max(1, width // 5)] *= 8.0
    return randn(tokens, width) * channel * torch.exp(0.3 * randn(tokens, 1))


def _pad(x, multiple):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % multiple))


def _rows8(x):
    """Rows in 8 bits with a scale per row and 128 columns, laid out as the package keeps them: rows of whole 16 bytes, scales
    with the rows next to each other."""
    tokens, width = x.shape
    b = _pad(x, BLOCK).view(tokens, -1, BLOCK)
    scale = b.abs().amax(-1).clamp_min(SMALLEST) / E4M3_MAX
    q = (b / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(tokens, -1)[:, :width]
    return _pad(q, 16).to(torch.float8_e4m3fn)[:, :width], scale.t().contiguous().t()


def _weight8(w):
    """A weight in 8 bits with a scale per 128 x 128 block."""
    rows, width = w.shape
    b = torch.nn.functional.pad(w, (0, -width % BLOCK, 0, -rows % BLOCK))
    b = b.view(b.shape[0] // BLOCK, BLOCK, b.shape[1] // BLOCK, BLOCK)
    scale = b.abs().amax((1, 3)).clamp_min(SMALLEST) / E4M3_MAX
    q = (b / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(b.shape[0] * BLOCK, -1)[:rows, :width]
    return _pad(q, 16).to(torch.float8_e4m3fn)[:, :width], scale


def prepare(case, seed):
    randn = _random(seed)
    tokens, width, op = case["tokens"], case["width"], case["op"]
    state = {"case": case}
    if op == "norm":
        dtype = DTYPES[case["dtype"]]
        state["x"] = _tokens(randn, tokens, width).to(dtype)
        state["branch"] = (2.0 * randn(tokens, width)).to(dtype)
        state["scale"] = (0.3 + 0.1 * randn(width)).to(dtype)
        norm = torch.nn.RMSNorm(width, eps=1e-6, device="cuda", dtype=dtype).requires_grad_(False)
        norm.weight.copy_(1.0 + 0.2 * randn(width))
        state["norm"] = norm
        return state
    x = _tokens(randn, tokens, width)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True))
    names = ("gate", "up") if op in ("gated", "gated8") else ("weight",)
    dtype = DTYPES.get(case["dtype"], torch.bfloat16)
    for name in names:
        w = randn(case["out"], width) * (1.5 / math.sqrt(width))
        bias = 0.2 * randn(case["out"]) if case["bias"] else None
        state[name] = _weight8(w) if op.endswith("8") else w.to(dtype)
        # 8-bit products take their bias in float32 (it is added to the float32 sums), 16-bit ones in the tokens' type
        state[name + "_bias"] = bias if bias is None or op.endswith("8") else bias.to(dtype)
    if op.endswith("8"):
        state["x"] = _rows8(x)
        return state
    state["x"] = x.to(dtype)
    if case["train"]:
        state["grad"] = randn(tokens, case["out"]).to(dtype)
        for name in ("x", "gate", "up", "gate_bias", "up_bias"):
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------
def _values(q, scale):
    """What 8-bit rows stand for, float32 (scale per row and 128 columns)."""
    return q.float() * scale.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _weight_values(q, scale):
    return q.float() * scale.repeat_interleave(BLOCK, 0)[: q.shape[0]].repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _quantized(y):
    """Values -> (8-bit numbers, their scale per row and 128 columns)."""
    rows, width = y.shape
    b = _pad(y, BLOCK).view(rows, -1, BLOCK)
    scale = b.abs().amax(-1).clamp_min(SMALLEST) / E4M3_MAX
    q = (b / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.reshape(rows, -1)[:, :width].to(torch.float8_e4m3fn), scale


def _activation(g, act):
    """(act(g), its derivative)"""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain(state):
    case = state["case"]
    op, dtype = case["op"], DTYPES.get(case["dtype"])
    if op == "norm":
        stream = (state["x"].float() + state["branch"].float() * state["scale"].float()).to(dtype)
        s = stream.float()
        y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + state["norm"].eps) * state["norm"].weight.float()
        if case["eight"]:
            values, scale = _quantized(y)
            return {"stream": stream, "values": values, "scale": scale}
        return {"stream": stream, "normed": y.to(dtype)}
    if op == "linear8":
        out = _values(*state["x"]) @ _weight_values(*state["weight"]).t()
        return {"out": (out if state["weight_bias"] is None else out + state["weight_bias"]).to(dtype)}
    if op == "gated8":
        x = _values(*state["x"])
        g, u = x @ _weight_values(*state["gate"]).t(), x @ _weight_values(*state["up"]).t()
        if case["bias"]:
            g, u = g + state["gate_bias"], u + state["up_bias"]
        h = _activation(g, case["act"])[0] * u
        if dtype is not None:
            return {"h": h.to(dtype)}
        values, scale = _quantized(h)
        return {"values": values, "scale": scale}
    with torch.no_grad():
        x, wg, wu = state["x"].float(), state["gate"].float(), state["up"].float()
        g, u = x @ wg.t(), x @ wu.t()
        if case["bias"]:
            g, u = g + state["gate_bias"].float(), u + state["up_bias"].float()
        a, slope = _activation(g, case["act"])
        out = {"h": (a * u).to(dtype)}
        if case["train"]:
            dh = state["grad"].float()
            dg, du = dh * u * slope, dh * a
            out["dx"] = (dg @ wg + du @ wu).to(dtype)
            out["dgate"], out["dup"] = (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype)
            if case["bias"]:
                out["dgate_bias"], out["dup_bias"] = dg.sum(0).to(dtype), du.sum(0).to(dtype)
        return out


def _own(state):
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import BlockScaled, block_scaled_gated_linear, block_scaled_linear
    from come_b200.feed_forward import gated_linear
    case = state["case"]
    op, dtype = case["op"], DTYPES.get(case["dtype"])
    if op == "norm":
        stream, normed = residual_rmsnorm(state["x"], state["branch"], state["scale"], state["norm"], quantize=case["eight"])
        if case["eight"]:
            return {"stream": stream, "values": normed.data, "scale": normed.scale}
        return {"stream": stream, "normed": normed}
    if op == "linear8":
        return {"out": block_scaled_linear(BlockScaled(*state["x"]), BlockScaled(*state["weight"]), state["weight_bias"], out_dtype=dtype)}
    if op == "gated8":
        h = block_scaled_gated_linear(BlockScaled(*state["x"]), BlockScaled(*state["gate"]), BlockScaled(*state["up"]), state["gate_bias"],
                                      state["up_bias"], activation=case["act"], out_dtype=dtype)
        return {"h": h} if dtype is not None else {"values": h.data, "scale": h.scale}
    leaves = {"dx": state["x"], "dgate": state["gate"], "dup": state["up"], "dgate_bias": state["gate_bias"], "dup_bias": state["up_bias"]}
    h = gated_linear(state["x"], state["gate"], state["up"], state["gate_bias"], state["up_bias"], activation=case["act"])
    if not case["train"]:
        return {"h": h}
    leaves = {name: leaf for name, leaf in leaves.items() if leaf is not None}
    return {"h": h.detach(), **dict(zip(leaves, torch.autograd.grad(h, list(leaves.values()), state["grad"])))}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    T, C, op = case["tokens"], case["width"], case["op"]
    size = {"f32": 4, "e4m3": 1}.get(case["dtype"], 2)
    blocks = lambda n: -(-n // BLOCK)  # noqa: E731
    if op == "norm":
        out = T * (C + 4 * blocks(C)) if case["eight"] else T * C * size
        return {"bytes": 3 * T * C * size + out + 2 * C * size, "flops": 7 * T * C}
    F = case["out"]
    bias = F * (4 if op.endswith("8") else size) if case["bias"] else 0
    if op in ("linear8", "gated8"):
        n = 2 if op == "gated8" else 1
        read = T * C + 4 * T * blocks(C) + n * (F * C + 4 * blocks(F) * blocks(C) + bias)
        write = T * F * size + (4 * T * blocks(F) if size == 1 else 0)
        return {"bytes": read + write, "flops": 2 * n * T * C * F}
    forward = T * C + 2 * F * C + T * F
    if not case["train"]:
        return {"bytes": forward * size + 2 * bias, "flops": 4 * T * C * F}
    # the step: reads the tokens, the weights and the result's gradient, writes the result and the gradients
    return {"bytes": (2 * T * C + 4 * F * C + 2 * T * F) * size + 4 * bias, "flops": 12 * T * C * F}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _exact_blocks(y):
    """Blocks of 128 columns scaled to a largest magnitude of 448 and rounded to 4 significant bits -> (scaled values, scales)."""
    values, scales = [], []
    for part in y.split(BLOCK, dim=1):
        largest = part.abs().max(dim=1).values
        scale = torch.maximum(largest, torch.full_like(largest, SMALLEST)) / 448
        z = part / scale.unsqueeze(1)
        # e4m3: normal numbers from 2^-6 up have 3 bits behind the leading one, below that the step stays 2^-9
        exponent = torch.frexp(z).exponent.clamp(min=-5) - 1
        step = torch.ldexp(torch.ones_like(z), exponent - 3)
        values.append((torch.round(z / step) * step).clamp(-448, 448))
        scales.append(scale)
    return torch.cat(values, 1), torch.stack(scales, 1)


def _wide(data, scale, rows_per_scale):
    wide = data.to(torch.float64)
    for i in range(scale.shape[1]):
        per_row = scale[:, i].to(torch.float64)
        if rows_per_scale > 1:
            per_row = per_row[torch.arange(data.shape[0], device=data.device) // rows_per_scale]
        wide[:, i * BLOCK: (i + 1) * BLOCK] *= per_row.unsqueeze(1)
    return wide


def exact(case, seed):
    state = prepare(case, seed)
    op, wide = case["op"], lambda t: t.detach().to(torch.float64)  # noqa: E731
    if op == "norm":
        stream = torch.addcmul(wide(state["x"]), wide(state["branch"]), wide(state["scale"]))
        stored = wide(stream.to(DTYPES[case["dtype"]]))  # the norm is that of the stream as it is stored
        y = wide(state["norm"].weight) * stored / torch.sqrt(stored.pow(2).mean(dim=1, keepdim=True) + state["norm"].eps)
        if not case["eight"]:
            return {"stream": stream, "normed": y}
        values, scale = _exact_blocks(y)
        return {"stream": stream, "values": values, "scale": scale}
    if op == "linear8":
        bias = 0.0 if state["weight_bias"] is None else wide(state["weight_bias"])
        return {"out": torch.einsum("tk,nk->tn", _wide(*state["x"], 1), _wide(*state["weight"], BLOCK)) + bias}
    zero = torch.zeros(case["out"], dtype=torch.float64, device="cuda")
    bg, bu = ((wide(state[n]) if case["bias"] else zero) for n in ("gate_bias", "up_bias"))
    x = _wide(*state["x"], 1) if op == "gated8" else wide(state["x"])
    wg, wu = ((_wide(*state[n], BLOCK) if op == "gated8" else wide(state[n])) for n in ("gate", "up"))
    g, u = torch.einsum("tk,fk->tf", x, wg) + bg, torch.einsum("tk,fk->tf", x, wu) + bu
    if case["act"] == "silu":
        s = torch.sigmoid(g)
        a, slope = g * s, s + g * s * torch.sigmoid(-g)
    else:
        tail = torch.special.erfc(-g / math.sqrt(2)) / 2
        a, slope = g * tail, tail + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
    h = a * u
    if op == "gated8":
        if case["dtype"] != "e4m3":
            return {"h": h}
        values, scale = _exact_blocks(h)
        return {"values": values, "scale": scale}
    out = {"h": h}
    if case["train"]:
        dh = wide(state["grad"])
        dg, du = dh * u * slope, dh * a
        out["dx"] = torch.einsum("tf,fk->tk", dg, wg) + torch.einsum("tf,fk->tk", du, wu)
        out["dgate"], out["dup"] = torch.einsum("tf,tk->fk", dg, x), torch.einsum("tf,tk->fk", du, x)
        if case["bias"]:
            out["dgate_bias"], out["dup_bias"] = dg.sum(dim=0), du.sum(dim=0)
    return out
