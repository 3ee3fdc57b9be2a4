"""Timed cases of the 8-bit path with block scales: rounding of activations and weights to e4m3,
RMSNorm and SwiGLU that end in it, and the matrix products of what comes out.

Kinds of case:

  quant    quantize_fp8_blocks: rows to e4m3, one fp32 scale for each 1 x 128 block (activations) or each
           128 x 128 block (weights)
  norm     rmsnorm_fp8_blocks: the residual's addition, RMSNorm and the rounding
  silu     silu_mul_fp8_blocks: SwiGLU of the two halves of a gate_up result, and the rounding
  linear   linear_fp8_blocks: e4m3 activations times e4m3 weights, each with its block scales
  grouped  grouped_linear_fp8_blocks: the same with one weight matrix for each group of rows (experts)

With a the largest |v| of a block, at least 2^-100, its scale is a / 448 in fp32 and its codes are the e4m3 values
nearest to 448 v / a, ties to even.  The last block of a row is shorter where the row is no multiple of 128.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 128
EPS = 1e-6
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}

_ops = None


def _framework():
    global _ops
    if _ops is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-deepseek-v2-lite_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from triton_kernels import fp8_blocks

        _ops = fp8_blocks
    return _ops


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # attention outputs of a batch of 64 before o_proj
        {"name": "quant_64", "kind": "quant", "rows": 64, "cols": 2048, "block": 1, "dtype": "bf16"},
        # the dense layer's gate_up weights, rounded once when a bf16 checkpoint is loaded
        {"name": "quant_weight", "kind": "quant", "rows": 21888, "cols": 2048, "block": 128, "dtype": "bf16"},
        # one chat's decode step
        {"name": "norm_1", "kind": "norm", "rows": 1, "cols": 2048, "residual": True, "dtype": "bf16"},
        # a chunk of prompts
        {"name": "norm_8192", "kind": "norm", "rows": 8192, "cols": 2048, "residual": True, "dtype": "bf16"},
        # the routes of 64 tokens to six experts each
        {"name": "silu_384", "kind": "silu", "rows": 384, "cols": 1408, "dtype": "bf16"},
        # the routes of a chunk of 8,192 tokens
        {"name": "silu_49152", "kind": "silu", "rows": 49152, "cols": 1408, "dtype": "bf16"},
        # one token's q | kv_a projection; the last scale block of the rows of weights is half a block
        {"name": "linear_1", "kind": "linear", "rows": 1, "out": 3648, "cols": 2048, "to": "bf16"},
        # five tokens' logits
        {"name": "linear_5_vocab", "kind": "linear", "rows": 5, "out": 102400, "cols": 2048, "to": "fp32"},
        # the dense layer's down projection of a batch of 64, with half a block at the end of each row
        {"name": "linear_64_down", "kind": "linear", "rows": 64, "out": 2048, "cols": 10944, "to": "bf16"},
        # the dense layer's gate_up projection of a chunk of prompts
        {"name": "linear_8192", "kind": "linear", "rows": 8192, "out": 21888, "cols": 2048, "to": "bf16"},
        # experts' gate_up at decode: 64 tokens, six of 64 experts each
        {"name": "grouped_64", "kind": "grouped", "tokens": 64, "groups": 64, "top": 6, "out": 2816, "cols": 2048,
         "gather": True, "to": "bf16"},
        # experts' gate_up for a chunk of prompts
        {"name": "grouped_8192", "kind": "grouped", "tokens": 8192, "groups": 64, "top": 6, "out": 2816, "cols": 2048,
         "gather": True, "to": "bf16"},
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi), spread over its logarithm."""
    return min(hi - 1, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cols(rng, lo, hi):
    """Row lengths: whole blocks, whole 16s or any."""
    n = _log_int(rng, lo, hi)
    unit = rng.choice([128, 128, 16, 1])
    return max(unit, n // unit * unit)


def draw(rng):
    kind = rng.choice(["quant", "norm", "silu", "linear", "grouped"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "quant":
        cols = _cols(rng, 64, 16385)
        return {"kind": kind, "rows": _log_int(rng, 1, min(32769, 40_000_000 // cols)), "cols": cols,
                "block": rng.choice([1, 128]), "dtype": dtype}
    if kind == "norm":
        cols = _cols(rng, 64, 12289)
        return {"kind": kind, "rows": _log_int(rng, 1, min(8193, 16_000_000 // cols)), "cols": cols,
                "residual": rng.random() < 0.7, "dtype": dtype}
    if kind == "silu":
        cols = _cols(rng, 64, 12289)
        return {"kind": kind, "rows": _log_int(rng, 1, min(49153, 60_000_000 // cols)), "cols": cols, "dtype": dtype}
    if kind == "linear":
        cols = _cols(rng, 64, 12289)
        out = _log_int(rng, 16, min(32769, 2 ** 27 // cols))
        most = min(8193, 2 ** 38 // (cols * out), 2 ** 27 // out)
        return {"kind": kind, "rows": _log_int(rng, 1, max(2, most)), "out": out, "cols": cols,
                "to": rng.choice(["bf16", "bf16", "fp32"])}
    groups = rng.choice([2, 8, 16, 60, 64, 64, 160])
    top = rng.randint(1, min(8, groups))
    cols = _cols(rng, 64, 4097)
    out = _log_int(rng, 32, min(4097, 360_000_000 // (groups * cols)))
    most = min(8193, 2 ** 37 // (cols * out * top))
    return {"kind": kind, "tokens": _log_int(rng, 1, max(2, most)), "groups": groups, "top": top, "out": out,
            "cols": cols, "gather": rng.random() < 0.6, "to": "bf16"}


def work(case):
    kind, cols = case["kind"], case["cols"]
    nb = -(-cols // BLOCK)
    if kind == "quant":
        rows, size = case["rows"], 2 if case["dtype"] == "bf16" else 4
        return {"bytes": rows * cols * (size + 1) + 4 * nb * -(-rows // case["block"]), "flops": 3 * rows * cols}
    if kind == "norm":
        rows, size = case["rows"], 2 if case["dtype"] == "bf16" else 4
        moved = 3 if case["residual"] else 1  # the input; with a residual that and the sum
        return {"bytes": rows * cols * (moved * size + 1) + cols * size + 4 * nb * rows, "flops": 8 * rows * cols}
    if kind == "silu":
        rows, size = case["rows"], 2 if case["dtype"] == "bf16" else 4
        return {"bytes": rows * cols * (2 * size + 1) + 4 * nb * rows, "flops": 9 * rows * cols}
    out, size = case["out"], 2 if case["to"] == "bf16" else 4
    matrix = out * cols + 4 * nb * -(-out // BLOCK)
    if kind == "linear":
        rows = case["rows"]
        return {"bytes": rows * (cols + 4 * nb) + matrix + rows * out * size, "flops": 2 * rows * out * cols}
    routes = case["tokens"] * case["top"]
    read = case["tokens"] if case["gather"] else routes
    hit = case["groups"] * (1 - (1 - case["top"] / case["groups"]) ** case["tokens"])  # groups that have rows
    return {"bytes": int(read * (cols + 4 * nb) + hit * matrix + routes * (out * size + 4)),
            "flops": 2 * routes * out * cols}


# ---------------------------------------------------------------- inputs
def _hidden(rows, cols, g, dtype):
    """Activations: channels of unequal size, a few of them far larger than the rest."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    gain = torch.exp(0.6 * torch.randn(cols, device=DEV, generator=g))
    gain = torch.where(torch.rand(cols, device=DEV, generator=g) < 0.004, gain * 20, gain)
    return (x * gain).to(dtype)


def _weight(rows, cols, g):
    """Weight codes and scales: rows of unequal size."""
    w = torch.randn(rows, cols, device=DEV, generator=g)
    w *= 0.02 * torch.exp(0.3 * torch.randn(rows, 1, device=DEV, generator=g))
    return _round_blocks(w, BLOCK)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, cols = case["kind"], case["cols"]
    s = {"kind": kind}
    if kind == "quant":
        s["x"] = _hidden(case["rows"], cols, g, TYPES[case["dtype"]])
        s["block"] = case["block"]
    elif kind == "norm":
        dtype = TYPES[case["dtype"]]
        s["x"] = _hidden(case["rows"], cols, g, dtype)
        s["residual"] = _hidden(case["rows"], cols, g, dtype) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(dtype)
    elif kind == "silu":
        both = 1.5 * torch.randn(case["rows"], 2 * cols, device=DEV, generator=g)
        s["gate_up"] = both.to(TYPES[case["dtype"]])
    elif kind == "linear":
        s["x"], s["x_scales"] = _round_blocks(_hidden(case["rows"], cols, g, torch.float32), 1)
        s["w"], s["w_scales"] = _weight(case["out"], cols, g)
        s["to"] = TYPES[case["to"]]
    else:
        groups, top, tokens, out = case["groups"], case["top"], case["tokens"], case["out"]
        score = torch.randn(tokens, groups, device=DEV, generator=g)
        score += 0.25 * torch.randn(groups, device=DEV, generator=g)  # some experts are asked more often
        group = score.topk(top, dim=1).indices.reshape(-1)
        order = torch.sort(group, stable=True).indices
        counts = torch.bincount(group, minlength=groups)
        s["offsets"] = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)]).to(torch.int32)
        s["most"] = int(counts.max())  # the largest group, for the plain form's padded batch
        s["rows"] = (order // top).to(torch.int32) if case["gather"] else None
        n = tokens if case["gather"] else tokens * top
        s["x"], s["x_scales"] = _round_blocks(_hidden(n, cols, g, torch.float32), 1)
        w, ws = _weight(groups * -(-out // BLOCK) * BLOCK, cols, g)  # each group begins a row of blocks
        s["w"] = w.view(torch.uint8).unflatten(0, (groups, -1))[:, :out].contiguous().view(E4M3)
        s["w_scales"] = ws.unflatten(0, (groups, -1)).contiguous()
        s["to"] = TYPES[case["to"]]
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    kind = s["kind"]
    if own:
        ops = _framework()
        if kind == "quant":
            return ops.quantize_fp8_blocks(s["x"], s["block"])
        if kind == "norm":
            return ops.rmsnorm_fp8_blocks(s["x"], s["weight"], EPS, s["residual"])
        if kind == "silu":
            gate, up = s["gate_up"].chunk(2, dim=1)
            return ops.silu_mul_fp8_blocks(gate, up)
        if kind == "linear":
            return ops.linear_fp8_blocks(s["x"], s["x_scales"], s["w"], s["w_scales"], s["to"])
        return ops.grouped_linear_fp8_blocks(s["x"], s["x_scales"], s["w"], s["w_scales"], s["offsets"], s["rows"],
                                             s["to"])
    if kind == "quant":
        return _round_blocks(s["x"].float(), s["block"])
    if kind == "norm":
        return _norm(s["x"], s["weight"], s["residual"])
    if kind == "silu":
        gate, up = s["gate_up"].float().chunk(2, dim=1)
        return _round_blocks(gate / (1 + torch.exp(-gate)) * up, 1)
    if kind == "linear":
        return (_values(s["x"], s["x_scales"], 1) @ _values(s["w"], s["w_scales"], BLOCK).T).to(s["to"])
    return _grouped(s)


# ---------------------------------------------------------------- plain forms
def _round_blocks(x, rows):
    """fp32 x [m, k] to e4m3 codes and the scales of its blocks of `rows` rows and 128 columns."""
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // BLOCK)
    if mb * rows > m or kb * BLOCK > k:
        y = x.new_zeros(mb * rows, kb * BLOCK)
        y[:m, :k] = x
    else:
        y = x
    y = y.view(mb, rows, kb, BLOCK)
    most = y.abs().amax((1, 3)).clamp(min=2.0 ** -100)
    codes = (y * 448 / most[:, None, :, None]).view(mb * rows, kb * BLOCK)[:m, :k]
    return codes.to(E4M3).contiguous(), most / 448


def _values(codes, scales, rows):
    """The fp32 values of codes [.., m, k] with scales [.., m / rows, k / 128]."""
    m, k = codes.shape[-2:]
    if rows > 1:
        scales = scales.repeat_interleave(rows, -2)[..., :m, :]
    return codes.float() * scales.repeat_interleave(BLOCK, -1)[..., :k]


def _norm(x, weight, residual):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * weight.float()
    return (*_round_blocks(y, 1), *(() if residual is None else (h,)))


def _grouped(s):
    """The rows laid out group by group, each padded to the largest, times the groups' weights."""
    offsets = s["offsets"].long()
    n = int(s["rows"].numel()) if s["rows"] is not None else s["x"].shape[0]
    x = _values(s["x"], s["x_scales"], 1)
    r = torch.arange(n, device=x.device)
    group = torch.searchsorted(offsets[1:].contiguous(), r, right=True)
    place = group * s["most"] + r - offsets[group]
    groups, out, k = s["w"].shape
    padded = x.new_zeros(groups * s["most"], k)
    padded[place] = x if s["rows"] is None else x[s["rows"].long()]
    w = _values(s["w"], s["w_scales"], BLOCK)
    y = torch.bmm(padded.view(groups, s["most"], k), w.transpose(1, 2))
    return y.view(-1, out)[place].to(s["to"])


# ---------------------------------------------------------------- in 64 bits
def _nearest_e4m3(v):
    """The e4m3 value nearest to each v, ties to the even one: steps of 2^(e - 3), e the exponent, at least -6."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    e = torch.where(torch.exp2(e) > v.abs().clamp(min=2.0 ** -6), e - 1, e)  # log2 rounds up next to a power
    step = torch.exp2(e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_blocks(y, rows):
    """(codes as values, scales)."""
    m, k = y.shape
    mb, kb = -(-m // rows), -(-k // BLOCK)
    at = (torch.arange(m, device=y.device) // rows)[:, None] * kb + torch.arange(k, device=y.device) // BLOCK
    most = torch.zeros(mb * kb, dtype=torch.float64, device=y.device)
    most.scatter_reduce_(0, at.reshape(-1), y.abs().reshape(-1), "amax")
    most = torch.maximum(most, torch.full_like(most, 2.0 ** -100))
    return _nearest_e4m3(y * 448 / most[at]), (most / 448).view(mb, kb)


def _exact_values(codes, scales, rows):
    m, k = codes.shape
    i, j = torch.arange(m, device=codes.device) // rows, torch.arange(k, device=codes.device) // BLOCK
    return codes.double() * scales.double()[i[:, None], j]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_blocks(s["x"].double(), case["block"])
    if kind == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = (h + s["residual"].double()).to(s["x"].dtype).double()
        # a row's factor cancels from 448 v / a: without it products of bf16 values, ties among them, are exact
        codes, scales = _exact_blocks(h * s["weight"].double(), 1)
        scales = scales / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS)
        return codes, scales, *(() if s["residual"] is None else (h,))
    if kind == "silu":
        n = case["cols"]
        gate, up = s["gate_up"][:, :n].double(), s["gate_up"][:, n:].double()
        return _exact_blocks(gate * torch.sigmoid(gate) * up, 1)
    if kind == "linear":
        return torch.matmul(_exact_values(s["x"], s["x_scales"], 1),
                            _exact_values(s["w"], s["w_scales"], BLOCK).t().contiguous())
    at = s["offsets"].tolist()
    parts = []
    for e in range(case["groups"]):
        if at[e + 1] > at[e]:
            x, xs = s["x"], s["x_scales"]
            mine = torch.arange(at[e], at[e + 1], device=DEV)
            mine = mine if s["rows"] is None else s["rows"][mine].long()
            x = x.view(torch.uint8)[mine].view(E4M3)
            w = _exact_values(s["w"][e], s["w_scales"][e], BLOCK)
            parts.append(torch.matmul(_exact_values(x, xs[mine], 1), w.t().contiguous()))
    return torch.cat(parts)
