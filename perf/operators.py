"""Workloads of the read-out operators: layer norm over looked-up rows, 8-bit activation checkpoints, and the
backward passes that read them.

A lookup hands a layer ``[tokens, entries_per_token * hidden]`` values: bf16, or e4m3 codes with one fp32 scale per
128 columns.  The model's read-out normalises them and projects them; training keeps the normalised rows in 8 bits
(e4m3 codes, power-of-two scales per 128 columns) and both the norm's and the projection's backward pass read that
one checkpoint.  ``run`` computes each operator from elementary torch operations, or, with ``own``, by the calls of
:mod:`engram_rdma_lab_b200.ops`.

Operators (``case["op"]``):

* ``norm``: layer norm of ``tokens`` rows, forward only (serving, or evaluation);
* ``train``: its forward and backward pass; ``keep`` says what is kept between them ("exact": the rows themselves,
  "fp8": the normalised rows in 8 bits);
* ``save``: activations to 8 bits and back;
* ``wgrad``: a projection's weight and bias gradients, from the gradient of its output and the 8-bit checkpoint of
  its input; with ``fold`` the checkpoint holds a norm's normalised rows and the projection's input was
  ``rows * norm_weight + norm_bias``.
"""

import math

import torch

own = False

BLOCK = 128  # columns of one scale
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# The largest listed cases; drawn ones stay within them.
MOST_TOKENS, MOST_WIDTH, MOST_OUT = 8192, 12288, 2048


def listed():
    return [
        # One decoded token's looked-up rows in a serving step: latency.
        {"name": "norm 1 token fp8 rows", "op": "norm", "tokens": 1, "ept": 24, "hidden": 256, "rows": "e4m3", "params": "bf16"},
        # One layer of a full lookup of 4096 tokens x 24 rows of 256 e4m3 values.
        {"name": "norm 4096 tokens fp8 rows", "op": "norm", "tokens": 4096, "ept": 24, "hidden": 256, "rows": "e4m3", "params": "bf16"},
        # Evaluation in fp32 at a width that no vector access divides.
        {"name": "norm 777x1001 fp32", "op": "norm", "tokens": 777, "ept": 1, "hidden": 1001, "rows": "fp32", "params": "fp32"},
        # A training step over bf16 tables, nothing rounded in between; fp32 parameters.
        {"name": "train 4096x6144 bf16", "op": "train", "tokens": 4096, "ept": 24, "hidden": 256, "rows": "bf16", "params": "fp32", "keep": "exact"},
        # The widest table set (24 rows of 512), kept in 8 bits.
        {"name": "train 8192x12288 bf16 fp8", "op": "train", "tokens": 8192, "ept": 24, "hidden": 512, "rows": "bf16", "params": "bf16", "keep": "fp8"},
        # A small table set (4 rows of 64) at 128 tokens, fp16.
        {"name": "train 128x256 fp16", "op": "train", "tokens": 128, "ept": 4, "hidden": 64, "rows": "fp16", "params": "fp16", "keep": "exact"},
        # Training straight from looked-up e4m3 rows.
        {"name": "train 4096 tokens fp8 rows", "op": "train", "tokens": 4096, "ept": 24, "hidden": 256, "rows": "e4m3", "params": "bf16", "keep": "fp8"},
        # A short batch's activations.
        {"name": "save 33x6144 fp16", "op": "save", "tokens": 33, "width": 6144, "dtype": "fp16"},
        # A full batch's activations.
        {"name": "save 8192x12288 bf16", "op": "save", "tokens": 8192, "width": 12288, "dtype": "bf16"},
        # A short, ragged batch of a small projection, fp32 gradients.
        {"name": "wgrad 100x256 to 72 fp32", "op": "wgrad", "tokens": 100, "width": 256, "out": 72, "dtype": "fp32", "fold": False},
        # The read-out's projection behind its norm at the full lookup of 4096 tokens.
        {"name": "wgrad 4096x6144 to 2048 norm", "op": "wgrad", "tokens": 4096, "width": 6144, "out": 2048, "dtype": "bf16", "fold": True},
        # A projection of the widest rows.
        {"name": "wgrad 8192x12288 to 2048", "op": "wgrad", "tokens": 8192, "width": 12288, "out": 2048, "dtype": "bf16", "fold": False},
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is evenly spread."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "train", "train", "save", "wgrad", "wgrad"])
    tokens = _spread(rng, 1, MOST_TOKENS)
    if op in ("norm", "train"):
        rows = rng.choice(["e4m3", "bf16", "bf16", "fp16", "fp32"])
        if rows == "e4m3" or rng.random() < 0.5:
            ept, hidden = rng.randint(1, 24), rng.choice([16, 64, 80, 128, 256, 256, 512])
        else:
            # The gradient of one or two columns is zero but for eps: nothing to compare.
            ept, hidden = 1, _spread(rng, 3 if op == "train" else 1, MOST_WIDTH)
        case = {"op": op, "tokens": tokens, "ept": ept, "hidden": hidden, "rows": rows}
        plain = "bf16" if rows == "e4m3" else rows
        case["params"] = rng.choice([plain, "fp32"])
        if op == "train":
            case["keep"] = "fp8" if rows == "e4m3" else rng.choice(["exact", "fp8"])
            if case["keep"] == "fp8":
                # One value that rounds the other way in 8 bits would show in an fp32 gradient.
                case["params"] = plain
                if rows == "fp32":
                    case["rows"] = case["params"] = "bf16"
            if case["rows"] == "fp32" and tokens * ept * hidden > MOST_TOKENS * MOST_WIDTH // 2:
                case["tokens"] = max(1, tokens // 2)
        return case
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "save":
        if dtype == "fp32":
            tokens = max(1, tokens // 2)
        return {"op": op, "tokens": tokens, "width": _spread(rng, 1, MOST_WIDTH), "dtype": dtype}
    if dtype != "bf16":  # more work for each product
        tokens = max(1, tokens // 4)
    return {"op": op, "tokens": tokens, "width": _spread(rng, 16, MOST_WIDTH), "out": _spread(rng, 8, MOST_OUT), "dtype": dtype,
            "fold": rng.random() < 0.5}


def _width(case):
    return case["width"] if "width" in case else case["ept"] * case["hidden"]


def _activations(g, m, n, dtype):
    """Residual-stream-like values: columns of different size, some with an offset, a few large ones."""
    scale = torch.exp2(torch.randn(n, generator=g, device="cuda"))
    offset = torch.randn(n, generator=g, device="cuda") * (torch.rand(n, generator=g, device="cuda") < 0.1) * 4
    x = torch.randn(m, n, generator=g, device="cuda")
    return x.mul_(scale).add_(offset).to(dtype)


def _lookup(g, m, ept, hidden):
    """What a lookup returns for e4m3 tables: codes, and scales laid out column by column with rows padded to 4.
    One entry in twenty is padding: zero rows with zero scales."""
    packs = -(-hidden // BLOCK)
    codes = torch.randn(m, ept, hidden, generator=g, device="cuda").clamp_(-448, 448)
    there = torch.rand(m, ept, 1, generator=g, device="cuda") >= 0.05
    codes = (codes * there).reshape(m, ept * hidden).to(torch.float8_e4m3fn)
    exponent = torch.randint(0, 9, (m, ept, packs), generator=g, device="cuda").float()
    values = (torch.exp2(-exponent) * there).reshape(m, ept * packs)
    padded = (m + 3) // 4 * 4
    scales = torch.zeros(ept * packs * padded, device="cuda").as_strided((m, ept * packs), (1, padded))
    scales.copy_(values)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    m, n, op = case["tokens"], _width(case), case["op"]
    state = dict(case)
    if op in ("norm", "train"):
        params = TYPES[case["params"]]
        if case["rows"] == "e4m3":
            state["x"], state["scales"] = _lookup(g, m, case["ept"], case["hidden"])
            out = torch.bfloat16
        else:
            out = TYPES[case["rows"]]
            state["x"], state["scales"] = _activations(g, m, n, out), None
        state["weight"] = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(params)
        state["bias"] = (0.2 * torch.randn(n, generator=g, device="cuda")).to(params)
        if op == "train":
            state["dy"] = (torch.randn(m, n, generator=g, device="cuda") * 0.05).to(out)
    elif op == "save":
        state["x"] = _activations(g, m, n, TYPES[case["dtype"]])
    else:
        x = torch.randn(m, n, generator=g, device="cuda")
        codes, scales = _to_8_bits(x)
        state["scales"] = scales
        # Rows of a checkpoint start on 16-byte boundaries.
        state["codes"] = torch.zeros(m, (n + 15) // 16 * 16, device="cuda").to(torch.float8_e4m3fn)[:, :n]
        state["codes"].copy_(codes)
        state["dy"] = (torch.randn(m, case["out"], generator=g, device="cuda") * 0.05).to(TYPES[case["dtype"]])
        state["norm_weight"] = state["norm_bias"] = None
        if case["fold"]:
            state["norm_weight"] = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(TYPES[case["dtype"]])
            state["norm_bias"] = (0.2 * torch.randn(n, generator=g, device="cuda")).to(TYPES[case["dtype"]])
    return state


# ---------------------------------------------------------------- plain forms
def _blocks(x):
    m, n = x.shape
    blocks = -(-n // BLOCK)
    return torch.nn.functional.pad(x, (0, blocks * BLOCK - n)).view(m, blocks, BLOCK)


def _to_8_bits(x):
    """e4m3 codes and the smallest power-of-two scales that bring each block within 448 = 0.875 * 2^9."""
    m, n = x.shape
    view = _blocks(x.float())
    largest = view.abs().amax(2)
    mantissa, exponent = torch.frexp(largest)
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)
    scales = torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), exponent), torch.ones_like(largest))
    codes = (view / scales[:, :, None]).to(torch.float8_e4m3fn)
    return codes.view(m, -1)[:, :n], scales


def _from_8_bits(codes, scales):
    m, n = codes.shape
    return (_blocks(codes.float()) * scales[:, :, None]).view(m, -1)[:, :n]


def _looked_up(x, scales, ept, hidden):
    """Rows as fp32 values; e4m3 rows of `hidden` columns each have a scale per 128 columns."""
    if scales is None:
        return x.float()
    m = x.shape[0]
    rows = x.float().view(m, ept, hidden)
    packs = scales.shape[1] // ept
    return (rows * scales.reshape(m, ept, packs).repeat_interleave(BLOCK, 2)[:, :, :hidden]).view(m, ept * hidden)


def _plain(s):
    op = s["op"]
    if op == "save":
        return _from_8_bits(*_to_8_bits(s["x"])).to(s["x"].dtype)
    if op == "wgrad":
        dy, rows = s["dy"].float(), _from_8_bits(s["codes"], s["scales"])
        if s["norm_weight"] is not None:
            rows = rows * s["norm_weight"].float() + s["norm_bias"].float()
        return (dy.t() @ rows).to(s["dy"].dtype), dy.sum(0).to(s["dy"].dtype)
    x = _looked_up(s["x"], s["scales"], s["ept"], s["hidden"])
    out = torch.bfloat16 if s["rows"] == "e4m3" else s["x"].dtype
    weight, bias = s["weight"].float(), s["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * weight + bias).to(out)
    if op == "norm":
        return y
    if s["keep"] == "fp8":
        hat = _from_8_bits(*_to_8_bits(hat))
    dy = s["dy"].float()
    g = dy * weight
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return y, dx.to(out), (dy * hat).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["bias"].dtype)


# ---------------------------------------------------------------- the framework's calls
def _own(s):
    from engram_rdma_lab_b200 import ops

    op = s["op"]
    if op == "save":
        codes, scales = ops.save_fp8(s["x"])
        return ops.restore_fp8(codes, scales, dtype=s["x"].dtype)
    if op == "wgrad":
        return ops.fp8_weight_grad(s["dy"], s["codes"], s["scales"], norm_weight=s["norm_weight"], norm_bias=s["norm_bias"])
    kwargs = {} if s["scales"] is None else {"scales": s["scales"], "hidden": s["hidden"]}
    y, kept = ops.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS, keep=s.get("keep"), **kwargs)
    if op == "norm":
        return y
    return (y, *ops.layer_norm_backward(s["dy"], kept, s["weight"]))


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    m, n, op = case["tokens"], _width(case), case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
    if op == "save":
        # In, codes out and back in, out: the codes are what the two calls exchange.
        return {"bytes": m * n * (2 * size[case["dtype"]] + 2), "flops": 4 * m * n}
    if op == "wgrad":
        e, o = size[case["dtype"]], case["out"]
        return {"bytes": m * n + 4 * m * -(-n // BLOCK) + e * (m * o + o * n + o) + (2 * n * e if case["fold"] else 0), "flops": 2 * m * n * o}
    rows, out = size[case["rows"]], size["bf16" if case["rows"] == "e4m3" else case["rows"]]
    scales = 4 * m * case["ept"] * -(-case["hidden"] // BLOCK) if case["rows"] == "e4m3" else 0
    total = m * n * (rows + out) + scales + 2 * n * size[case["params"]]
    if op == "norm":
        return {"bytes": total, "flops": 8 * m * n}
    return {"bytes": total + 2 * m * n * out + 2 * n * size[case["params"]], "flops": 20 * m * n}


# ---------------------------------------------------------------- 64 bits
def _e4m3(v):
    """float64 values to the nearest e4m3 value, ties to even (|v| <= 448)."""
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp_min(-6).double() - 3)
    return torch.round(v / step) * step


def _kept(v):
    """float64 rows as their 8-bit checkpoint holds them: per 128 columns the least s = 2^k with max|v| <= 448 s."""
    out = torch.empty_like(v)
    for at in range(0, v.shape[1], BLOCK):
        part = v[:, at:at + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        k = torch.ceil(torch.log2(top / 448))
        k = torch.where(top / 448 <= torch.exp2(k - 1), k - 1, k)  # log2 that came out above a whole number
        s = torch.where(top > 0, torch.exp2(k), torch.ones_like(top))
        out[:, at:at + BLOCK] = _e4m3(part / s) * s
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "save":
        return _kept(s["x"].double())
    if op == "wgrad":
        columns = torch.arange(case["width"], device="cuda") // BLOCK
        rows = s["codes"].double() * s["scales"].double()[:, columns]
        dy = s["dy"].double()
        if case["fold"]:
            rows = rows * s["norm_weight"].double()[None] + s["norm_bias"].double()[None]
        return torch.einsum("mo,mn->on", dy, rows), torch.einsum("mo->o", dy)
    x = s["x"].double()
    if s["scales"] is not None:
        column = torch.arange(x.shape[1], device="cuda")
        packs = -(-case["hidden"] // BLOCK)
        x = x * s["scales"].double()[:, column // case["hidden"] * packs + column % case["hidden"] // BLOCK]
    n = x.shape[1]
    mean = torch.einsum("mn->m", x) / n
    x = x - mean[:, None]
    deviation = torch.sqrt(torch.einsum("mn,mn->m", x, x) / n + EPS)
    x = x / deviation[:, None]
    weight = s["weight"].double()
    y = x * weight[None] + s["bias"].double()[None]
    if op == "norm":
        return y
    if case["keep"] == "fp8":
        x = _kept(x)
    dy = s["dy"].double()
    # dL/dx_j = (w_j dy_j - A - x_j B) / deviation, with the row's means A of w dy and B of w dy x.
    a = torch.einsum("n,mn->m", weight, dy) / n
    b = torch.einsum("n,mn,mn->m", weight, dy, x) / n
    dx = (dy * weight[None] - a[:, None] - x * b[:, None]) / deviation[:, None]
    return y, dx, torch.einsum("mn,mn->n", dy, x), torch.einsum("mn->n", dy)
