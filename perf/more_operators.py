"""Linear layers in microscaled 4-bit floating point, as cases that can be timed: rows quantized to blocks of 32 e2m1 codes that
share a power of two, and read back; the product of two such matrices; both projections of a gated feed-forward block with
their activation; and the products of a router's experts.

A case is a dict of plain values; `prepare` makes what a serving program holds before the call, `run` is one pass: with `own`
through the package's public entry points, without it in elementary torch operations in 32 bits, rounded once.
Activations are N(0, 1) as they leave a norm, one channel in a hundred scaled by 20; weights are N(0, 0.02).
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 32
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # magnitudes of the codes 0 ... 7; bit 3 is the sign


def _read_back(rows, k, dtype="bf16"):
    return {"kind": "read_back", "rows": rows, "k": k, "dtype": dtype}


def _mm(m, n, k, bias="none", dtype="bf16"):
    return {"kind": "mm", "m": m, "n": n, "k": k, "bias": bias, "dtype": dtype}


def _gated(m, n, k, dtype="bf16"):
    return {"kind": "gated", "m": m, "n": n, "k": k, "dtype": dtype}


def _experts(experts, rows, n, k, gated=False, even=False):
    return {"kind": "experts", "experts": experts, "m": rows, "n": n, "k": k, "gated": gated, "even": even}


def listed():
    named = {
        # One token's activations on their way into a layer: the smallest call there is, all latency.
        "read_back_1": _read_back(1, 4096),
        # The activations of a large prefill step between two layers.
        "read_back_8192": _read_back(8192, 28672),
        # One user, one new token: a square projection.
        "mm_1": _mm(1, 8192, 8192),
        # A decode batch on the second projection of a feed-forward block.
        "mm_64": _mm(64, 4096, 14336),
        # A ragged prefill step of a large model.
        "mm_500": _mm(500, 10240, 8192),
        # An ordinary square product.
        "mm_4096": _mm(4096, 4096, 4096),
        # A large prefill step through a wide projection with bias.
        "mm_8192_bias": _mm(8192, 28672, 4096, bias="bf16"),
        # The first half of a feed-forward block: a decode batch ...
        "gated_16": _gated(16, 14336, 4096),
        # ... and a prefill step of odd sizes, in fp16.
        "gated_2047_fp16": _gated(2047, 10000, 4128, dtype="fp16"),
        # A decode batch routed to 16 experts: the weights of all of them for a few rows each.
        "experts_256": _experts(16, 256, 5120, 4096, gated=True),
        # A prefill step over 16 experts, some of them crowded.
        "experts_8192": _experts(16, 8192, 8192, 5120),
        # Many small experts, the first half of their feed-forward blocks.
        "experts_128": _experts(128, 32768, 768, 2048, gated=True),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    """One more case: sizes spread over the logarithm of their range, odd ones among them."""
    kind = rng.choice(["read_back", "mm", "mm", "gated", "experts", "experts"])
    k = _BLOCK * _log_int(rng, 1, 512)
    if kind == "read_back":
        rows = _log_int(rng, 1, 32768)
        while rows > 1 and rows * k > 8192 * 28672 // 2:
            rows //= 2
        return _read_back(rows, k, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    n = rng.choice([1, 1, 8, 16, 64]) * _log_int(rng, 8, 4096)
    n = min(n, 28672)
    if kind == "experts":
        experts = _log_int(rng, 1, 128)
        case = _experts(experts, _log_int(rng, 1, 32768), n, k, rng.random() < 0.5, rng.random() < 0.2)
        limit = 128 * 8192 * 5120   # of all experts' weights
        while case["experts"] * case["n"] * case["k"] * (2 if case["gated"] else 1) > limit // 2:
            case["experts"] = max(1, case["experts"] // 2)
            case["n"] = max(8, int(0.8 * case["n"]))
        while _padded_flops(case) > 2 * 8192 * 28672 * 4096:
            case["m"] = max(1, int(0.7 * case["m"]))
        return case
    m = _log_int(rng, 1, 16384)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    case = _mm(m, n, k, rng.choice(["none", "none", "bf16", "fp32"]), dtype) if kind == "mm" else _gated(m, n, k, dtype)
    while work(case)["flops"] > 2 * 8192 * 28672 * 4096:
        case["m"] = max(1, int(0.7 * case["m"]))
    return case


# ---------------------------------------------------------------------------------------------------------------------
# rows per expert: part of a case, the same for every seed
# ---------------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """Rows of each expert: popularity falls with the rank as rank^-1.1, the ranks in any order; or the same for all."""
    experts, rows = case["experts"], case["m"]
    if case["even"]:
        return [rows // experts + (e < rows % experts) for e in range(experts)]
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    weights = [(e + 1) ** -1.1 for e in range(experts)]
    rng.shuffle(weights)
    sizes = [0] * experts
    for e in rng.choices(range(experts), weights, k=rows):
        sizes[e] += 1
    return sizes


def _padded_flops(case):
    return 2 * case["experts"] * max(_sizes(case)) * case["n"] * case["k"] * (2 if case["gated"] else 1)


def _stored(rows, k):
    """Bytes of rows of codes and their scales."""
    return rows * (k // 2 + k // _BLOCK)


def work(case):
    k = case["k"]
    if case["kind"] == "read_back":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": (size + 2) * case["rows"] * k + 2 * _stored(case["rows"], k), "flops": 0}
    m, n = case["m"], case["n"]
    wide = 2 * n if case["kind"] == "gated" or case.get("gated") else n   # rows of the weights
    used = sum(size > 0 for size in _sizes(case)) if case["kind"] == "experts" else 1
    return {"bytes": _stored(m, k) + used * _stored(wide, k) + 2 * m * n, "flops": 2 * m * wide * k}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _encode(x):
    """Rows in 32 bits -> packed codes [.., K / 2], the earlier value in the low half of a byte, and exponents + 127 [.., K / 32]."""
    blocks = x.unflatten(-1, (-1, _BLOCK))
    _, exponent = torch.frexp(blocks.abs().amax(-1, keepdim=True))   # amax in [2^(exponent - 1), 2^exponent)
    exponent = torch.where(blocks.abs().amax(-1, keepdim=True) == 0, -127, (exponent - 3).clamp(min=-127))
    v = blocks * torch.exp2(-exponent.float())
    a = v.abs()
    a = torch.where(a < 2, (2 * a).round() / 2, torch.where(a < 4, a.round(), 2 * (a / 2).round())).clamp(max=6.0)
    code = torch.where(a <= 2, 2 * a, torch.where(a <= 4, a + 2, a / 2 + 4)).to(torch.uint8)   # (place in _GRID)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), (exponent.squeeze(-1) + 127).to(torch.uint8)


def _decode(codes, scales):
    """What packed codes and their scales stand for, in 32 bits."""
    grid = torch.tensor(_GRID + tuple(-x for x in _GRID), device=codes.device)
    values = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).flatten(-2)
    power = torch.exp2(scales.float() - 127)
    return (values.unflatten(-1, (-1, _BLOCK)) * power[..., None]).flatten(-2)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind, k = case["kind"], case["k"]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    def activations(rows):
        x = normal(rows, k)
        x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 100)]] *= 20
        return x

    if kind == "read_back":
        return {"kind": kind, "x": activations(case["rows"]).to(_DTYPES[case["dtype"]])}
    m, n = case["m"], case["n"]
    state = {"kind": kind, "n": n, "dtype": _DTYPES[case.get("dtype", "bf16")], "gated": kind == "gated" or case.get("gated", False)}
    state["xq"], state["xs"] = _encode(activations(m).bfloat16().float())
    wide = 2 * n if state["gated"] else n
    if kind == "experts":
        parts = [_encode(normal(wide, k, std=0.02).bfloat16().float()) for _ in range(case["experts"])]
        state["wq"], state["ws"] = (torch.stack(p) for p in zip(*parts))
        sizes = _sizes(case)
        state.update(sizes=torch.tensor(sizes).cuda(), most=max(sizes))
        return state
    state["wq"], state["ws"] = _encode(normal(wide, k, std=0.02).bfloat16().float())
    state["bias"] = None if case.get("bias", "none") == "none" else normal(n, std=0.1).to(_DTYPES[case["bias"]])
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _activated(y):
    """silu of the first half of the columns times the second half."""
    gate, up = y.chunk(2, -1)
    return gate / (1 + torch.exp(-gate)) * up


def _plain(s):
    if s["kind"] == "read_back":
        return _decode(*_encode(s["x"].float())).to(torch.bfloat16)
    x, w = _decode(s["xq"], s["xs"]), _decode(s["wq"], s["ws"])
    if s["kind"] == "experts":   # the rows of an expert side by side, padded to the longest
        sizes = s["sizes"]
        first = sizes.cumsum(0) - sizes
        row = torch.arange(x.shape[0], device="cuda")
        expert = torch.searchsorted(first + sizes, row, right=True)
        at = (first[:, None] + torch.arange(s["most"], device="cuda")).clamp(max=x.shape[0] - 1)
        y = torch.bmm(x[at], w.transpose(1, 2).contiguous())[expert, row - first[expert]]
    else:
        y = torch.matmul(x, w.t())
        if s["bias"] is not None:
            y = y + s["bias"].float()
    if s["gated"]:
        y = _activated(y)
    return y.to(s["dtype"])


def run(state):
    s = state
    if not own:
        return _plain(s)
    import mslk_amd

    if s["kind"] == "read_back":
        return mslk_amd.dequantize_mxfp4(*mslk_amd.quantize_mxfp4(s["x"]))
    operands = (s["xq"], s["wq"], s["xs"], s["ws"])
    if s["kind"] == "experts":
        return mslk_amd.mxfp4_grouped_mm(*operands, s["sizes"], gated=s["gated"])
    if s["kind"] == "gated":
        return mslk_amd.mxfp4_gated_mm(*operands, out_dtype=s["dtype"])
    return mslk_amd.mxfp4_mm(*operands, bias=s["bias"], out_dtype=s["dtype"])


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_values(codes, scales):
    """The same as _decode, from the fields of the codes: (-1)^s 2^(e - 1) (1 + m / 2), for e = 0 (-1)^s m / 2."""
    nibbles = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = codes // 16 if half else codes % 16
        sign, field, low = 1.0 - 2.0 * (c // 8).double(), ((c % 8) // 2).double(), (c % 2).double()
        nibbles[..., half::2] = sign * torch.where(field == 0, low / 2, 2.0 ** (field - 1) * (1 + low / 2))
    return nibbles * (2.0 ** (scales.double() - 127)).repeat_interleave(_BLOCK, -1)


def _exact_read_back(x):
    """Every value to the nearest one of the block's grid; of two as near, the one of even place."""
    blocks = x.double().unflatten(-1, (-1, _BLOCK))
    largest = blocks.abs().amax(-1, keepdim=True)
    unit = torch.where(largest == 0, 1.0, 2.0 ** (torch.floor(torch.log2(torch.where(largest == 0, 1.0, largest))) - 2))
    v = blocks.abs() / unit
    out = torch.zeros_like(v)
    for place in range(1, len(_GRID)):
        middle = (_GRID[place - 1] + _GRID[place]) / 2
        out[(v >= middle) if place % 2 == 0 else (v > middle)] = _GRID[place]
    return (torch.copysign(out, blocks) * unit).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "read_back":
        return torch.cat([_exact_read_back(x) for x in s["x"].split(max(1, (1 << 26) // case["k"]))])
    parts, at = [], 0
    for e, rows in enumerate(_sizes(case) if case["kind"] == "experts" else [case["m"]]):
        if rows == 0:
            continue
        wq, ws = (s["wq"][e], s["ws"][e]) if case["kind"] == "experts" else (s["wq"], s["ws"])
        y = _exact_values(s["xq"][at:at + rows], s["xs"][at:at + rows]) @ _exact_values(wq, ws).t().contiguous()
        at += rows
        if s.get("bias") is not None:
            y += s["bias"].double()
        if s["gated"]:
            gate, up = y[:, : case["n"]], y[:, case["n"]:]
            y = gate * torch.sigmoid(gate) * up
        parts.append(y)
    return torch.cat(parts)
