"""The attention of a served decoder layer, as cases that can be timed: new keys and values rotated and appended to a paged
cache, the attention of one new token per sequence over that cache, and the causal attention of whole prompts packed one
after the other.

A case is a dict of plain values; `prepare` makes what a serving program holds before the call, `run` is one pass: with
`own` through the package's public entry points, without it in elementary torch operations in 32 bits, rounded once.
Queries, keys and values are N(0, 1) as normalised activations leave their projections, with one channel in a hundred of
the keys scaled by 8 where the cache is kept in FP8 (the outliers that row scales exist for).
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_FP8 = torch.float8_e4m3fn
_FP8_MAX = 448.0


def _append(tokens, sequences, hq, hkv, d, page, cache="same", dtype="bf16", past=2000, rotary=None, interleaved=False):
    return {"kind": "append", "tokens": tokens, "sequences": sequences, "hq": hq, "hkv": hkv, "d": d, "page": page, "cache": cache,
            "dtype": dtype, "past": past, "rotary": d if rotary is None else rotary, "interleaved": interleaved}


def _decode(sequences, longest, hq, hkv, d, page, cache="same", dtype="bf16", shortest=1):
    return {"kind": "decode", "sequences": sequences, "longest": longest, "shortest": shortest, "hq": hq, "hkv": hkv, "d": d,
            "page": page, "cache": cache, "dtype": dtype}


def _prompt(tokens, sequences, hq, hkv, d, dtype="bf16", causal=True, past=0):
    return {"kind": "prompt", "tokens": tokens, "sequences": sequences, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
            "causal": causal, "past": past}


def listed():
    named = {
        # One user, one new token: the smallest call there is, all latency.
        "append_1": _append(1, 1, 64, 8, 128, 16),
        # A decode batch, one token per sequence, on a cache kept in FP8.
        "append_64_fp8": _append(64, 64, 64, 8, 128, 16, cache="fp8"),
        # Prompts of several users packed together, as one prefill step appends them.
        "append_8191": _append(8191, 7, 64, 8, 128, 64, past=0),
        # One user in the middle of a conversation.
        "decode_1": _decode(1, 700, 32, 8, 128, 16, shortest=700),
        # A small batch without shared heads, small heads, fp16.
        "decode_8_fp16": _decode(8, 3001, 16, 16, 64, 16, dtype="fp16"),
        # An ordinary decode batch with lengths from nothing (a free place in the batch) to long.
        "decode_32": _decode(32, 8192, 64, 8, 128, 16, shortest=0),
        # One very long context: rows are few, the work lies along the cache.
        "decode_1_long": _decode(1, 131071, 64, 8, 128, 64, shortest=131071),
        # A large batch with a cache in FP8.
        "decode_128_fp8": _decode(128, 8192, 64, 8, 128, 64, cache="fp8", shortest=1000),
        # A short question, alone.
        "prompt_100": _prompt(100, 1, 32, 8, 128),
        # A prefill step of several users' prompts of very different lengths, a few of which continue a cached part.
        "prompt_packed": _prompt(8192, 9, 64, 8, 128, past=1000),
        # Texts to be embedded: no causal mask, heads of 96, fp16.
        "prompt_both_ways": _prompt(6000, 13, 16, 16, 96, dtype="fp16", causal=False),
        # One whole long document.
        "prompt_16384": _prompt(16384, 1, 32, 8, 128),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    """One more case: sizes spread over the logarithm of their range, odd ones among them."""
    hkv = rng.choice([1, 2, 4, 8, 8, 8, 16])
    hq = hkv * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 8) if hkv * g <= 64])
    d = rng.choice([64, 80, 96, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    if kind == "prompt":
        tokens = _log_int(rng, 1, 16384)
        sequences = min(tokens, _log_int(rng, 1, 64))
        case = _prompt(tokens, sequences, hq, hkv, d, dtype, rng.random() < 0.8, rng.choice([0, 0, _log_int(rng, 1, 2000)]))
        while _padded_scores(case) > 32 * 16384**2 or work(case)["flops"] > 2.2e12:
            case["tokens"] = max(1, int(0.8 * case["tokens"]))
            case["sequences"] = min(case["sequences"], case["tokens"])
        return case
    page = rng.choice([16, 16, 32, 64, 128])
    cache = rng.choice(["same", "same", "fp8"])
    if kind == "append":
        tokens = _log_int(rng, 1, 8191)
        sequences = rng.choice([tokens, _log_int(rng, 1, tokens)]) if tokens <= 512 else _log_int(rng, 1, 256)
        rotary = rng.choice([d, d, d // 2])
        case = _append(tokens, sequences, hq, hkv, d, page, cache, dtype, _log_int(rng, 1, 4000), rotary, rng.random() < 0.3)
        while case["tokens"] > 1 and case["tokens"] * (hq + 2 * hkv) * d > 8191 * 80 * 128:
            case["tokens"] = max(1, case["tokens"] // 2)
            case["sequences"] = min(case["sequences"], case["tokens"])
        return case
    sequences = _log_int(rng, 1, 256)
    longest = _log_int(rng, 1, 131072)
    case = _decode(sequences, longest, hq, hkv, d, page, cache, dtype, rng.choice([0, 1, max(1, longest // 2), longest]))
    while work(case)["bytes"] > 1.2e9 or case["sequences"] * case["longest"] * hkv * d > 128 * 8192 * 8 * 128:
        case["longest"] = max(1, case["longest"] // 2)
        case["shortest"] = min(case["shortest"], case["longest"])
    return case


# ---------------------------------------------------------------------------------------------------------------------
# lengths: part of a case, the same for every seed
# ---------------------------------------------------------------------------------------------------------------------
def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _split(rng, total, parts):
    """`parts` lengths of very different sizes that add up to `total`."""
    if parts == total:
        return [1] * parts
    cuts = [rng.expovariate(1.0) for _ in range(parts)]
    lengths = [int(total * c / sum(cuts)) for c in cuts]
    lengths[lengths.index(max(lengths))] += total - sum(lengths)
    return lengths


def _lengths(case):
    """(new tokens per sequence, length of each sequence's keys with them)."""
    rng = _rng(case)
    if case["kind"] == "decode":
        total = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["sequences"])]
        total[rng.randrange(len(total))] = case["longest"]
        if case["shortest"] == 0 and len(total) > 1:
            total[total.index(min(total))] = 0
        return [1] * len(total), total
    new = _split(rng, case["tokens"], case["sequences"])
    return new, [n + rng.randint(0, case["past"]) for n in new]


def _padded_scores(case):
    new, total = _lengths(case)
    return len(new) * case["hq"] * max(new) * max(total)


def _pairs(new, total, causal):
    """Query-key pairs that the mask leaves."""
    return sum(n * t - (n * (n - 1) // 2 if causal else 0) for n, t in zip(new, total))


def work(case):
    new, total = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "prompt":
        nq, nk = sum(new), sum(total)
        return {"bytes": 2 * d * (2 * nq * hq + 2 * nk * hkv) + 4 * nq * hq, "flops": 4 * hq * d * _pairs(new, total, case["causal"])}
    row = (d + 4) if case["cache"] == "fp8" else 2 * d   # a cached row: codes and their scale, or 16-bit values
    if case["kind"] == "append":
        nq = sum(new)
        return {"bytes": nq * (4 * hq * d + 4 * hkv * d + 2 * hkv * row + 4 * case["rotary"]), "flops": 3 * nq * (hq + hkv) * case["rotary"]}
    n = sum(total)
    return {"bytes": 2 * n * hkv * row + len(total) * hq * (4 * d + 4), "flops": 4 * n * hq * d}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32).cuda()


def _rotary_table(positions, rotary):
    """cos and sin of every position, side by side: [positions, rotary] in 32 bits, as a model computes it once."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def _quantize(x):
    """Rows in 32 bits -> e4m3 codes and one scale per row."""
    amax = x.abs().amax(-1, keepdim=True).clamp(min=1e-12)
    return (x * (_FP8_MAX / amax)).to(_FP8), (amax / _FP8_MAX).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    new, total = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    state = {"kind": case["kind"], "hq": hq, "hkv": hkv, "d": d, "max_new": max(new), "max_total": max(total)}
    if case["kind"] == "prompt":
        state.update(q=normal(sum(new), hq, d), k=normal(sum(total), hkv, d), v=normal(sum(total), hkv, d), cu_q=_offsets(new),
                     cu_k=_offsets(total) if new != total else None, causal=case["causal"], sequences=len(new))
        return state
    page = case["page"]
    pages = [-(-t // page) for t in total]
    pool = sum(pages) + 8
    ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)[: sum(pages)].cpu()
    table = torch.full((len(total), max(pages) + 3), -1, dtype=torch.int32)   # room to grow; no page where none is needed
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = ids[at:at + n]
        at += n
    state.update(page=page, table=table.cuda(), lens=torch.tensor(total, dtype=torch.int32).cuda(), k_scale=None, v_scale=None)
    if case["kind"] == "append":
        heads = normal(sum(new), hq + 2 * hkv, d)   # the fused projection's output; the three are views of it
        state.update(q=heads[:, :hq], k=heads[:, hq:hq + hkv], v=heads[:, hq + hkv:], cu_q=None if max(new) == min(new) == 1 else _offsets(new),
                     rotary=_rotary_table(max(total), case["rotary"]), interleaved=case["interleaved"])
        state.update(k_cache=torch.zeros(pool, page, hkv, d, device="cuda", dtype=_FP8 if case["cache"] == "fp8" else dtype))
        state.update(v_cache=torch.zeros_like(state["k_cache"]))
        if case["cache"] == "fp8":
            state.update(k_scale=torch.zeros(pool, page, hkv, device="cuda"), v_scale=torch.zeros(pool, page, hkv, device="cuda"))
        return state
    state.update(q=normal(len(total), hq, d), k_cache=normal(pool, page, hkv, d), v_cache=normal(pool, page, hkv, d))
    if case["cache"] == "fp8":
        loud = torch.randperm(d, generator=g, device="cuda")[: max(1, d // 100)]
        state["k_cache"][..., loud] *= 8
        for name in ("k", "v"):
            state[name + "_cache"], state[name + "_scale"] = _quantize(state[name + "_cache"].float())
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] channels of x [T, H, D] turned by their angles."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _append_plain(s):
    token = torch.arange(s["q"].shape[0], device="cuda")
    if s["cu_q"] is None:
        seq, position = token, s["lens"].long() - 1
    else:
        cu = s["cu_q"].long()
        seq = torch.searchsorted(cu[1:], token, right=True)
        position = s["lens"].long()[seq] - (cu[seq + 1] - token)
    page, slot = s["table"].long()[seq, position // s["page"]], position % s["page"]
    cos, sin = s["rotary"][position].chunk(2, -1)
    q = _rotate(s["q"].float(), cos, sin, s["interleaved"]).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, s["interleaved"])
    if s["k_scale"] is None:
        s["k_cache"][page, slot] = k.to(s["k_cache"].dtype)
        s["v_cache"][page, slot] = s["v"]
        return q, s["k_cache"], s["v_cache"]
    k, k_scale = _quantize(k)
    v, v_scale = _quantize(s["v"].float())
    s["k_cache"].view(torch.uint8)[page, slot] = k.view(torch.uint8)
    s["v_cache"].view(torch.uint8)[page, slot] = v.view(torch.uint8)
    s["k_scale"][page, slot] = k_scale
    s["v_scale"][page, slot] = v_scale
    return q, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _softmax_product(scores, masked, v):
    """exp(scores) v over the sum of exp(scores), and the sum's logarithm; zeros and -inf where everything is masked."""
    scores = scores.masked_fill_(masked, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / torch.where(total == 0, 1.0, total)
    return out, (total.log() + top).squeeze(-1)


def _decode_plain(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    sequences = s["q"].shape[0]
    table = s["table"].long().clamp(min=0)

    def rows(cache, scale):   # [B, Hkv, S, D]
        x = cache[table].float()
        if scale is not None:
            x = x * scale[table][..., None]
        return x.flatten(1, 2).transpose(1, 2).contiguous()

    k, v = rows(s["k_cache"], s["k_scale"]), rows(s["v_cache"], s["v_scale"])
    q = s["q"].float().view(sequences, hkv, hq // hkv, d) / math.sqrt(d)
    masked = torch.arange(k.shape[2], device="cuda") >= s["lens"][:, None]
    out, lse = _softmax_product(torch.matmul(q, k.transpose(2, 3)), masked[:, None, None], v)
    return out.reshape(sequences, hq, d).to(s["q"].dtype), lse.reshape(sequences, hq)


def _prompt_plain(s):
    hq, hkv, d, b = s["hq"], s["hkv"], s["d"], s["sequences"]
    nq, nk = s["max_new"], s["max_total"]
    cu_q = s["cu_q"].long()
    cu_k = cu_q if s["cu_k"] is None else s["cu_k"].long()
    i, j = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
    len_q, len_k = (cu_q[1:] - cu_q[:-1])[:, None], (cu_k[1:] - cu_k[:-1])[:, None]
    at_q = (cu_q[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)     # padded to the longest
    at_k = (cu_k[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    q = (s["q"].float() / math.sqrt(d))[at_q].view(b, nq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    k = s["k"].float()[at_k].permute(0, 2, 3, 1).contiguous()
    v = s["v"].float()[at_k].transpose(1, 2).contiguous()
    masked = (j >= len_k)[:, None, :].expand(b, nq, nk)
    if s["causal"]:
        masked = masked | (j > i[None, :, None] + (len_k - len_q)[:, :, None])
    scores = torch.matmul(q, k).view(b, hkv, hq // hkv, nq, nk)
    out, lse = _softmax_product(scores, masked[:, None, None], v[:, :, None])
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu_q[1:], token, right=True)
    place = token - cu_q[seq]
    return out[seq, :, :, place].reshape(-1, hq, d).to(s["q"].dtype), lse[seq, :, :, place].reshape(-1, hq)


def run(state):
    s = state
    if not own:
        return {"append": _append_plain, "decode": _decode_plain, "prompt": _prompt_plain}[s["kind"]](s)
    import mslk_amd

    if s["kind"] == "append":
        q = mslk_amd.append_kv(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], cu_seqlens=s["cu_q"],
                               rotary=s["rotary"], interleaved=s["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        held = (s["k_cache"], s["v_cache"])
        return (q, *held) if s["k_scale"] is None else (q, *held, s["k_scale"], s["v_scale"])
    if s["kind"] == "decode":
        return mslk_amd.attention_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], k_scale=s["k_scale"],
                                         v_scale=s["v_scale"], return_lse=True)
    return mslk_amd.attention_prompt(s["q"], s["k"], s["v"], s["cu_q"], cu_seqlens_k=s["cu_k"], causal=s["causal"], return_lse=True)


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------------------------------------------------
def _exact_rows(q, k, v, first, causal):
    """q [n, hq, d] at positions first, first + 1, ... over k, v [t, hkv, d]; a few rows at a time."""
    n, hq, d = q.shape
    t, hkv, _ = k.shape
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    if t == 0:
        return out, lse
    group = hq // hkv
    kt, vt = k.double().permute(1, 2, 0).contiguous(), v.double().transpose(0, 1).contiguous()
    step = max(1, (1 << 27) // (hq * t))
    for r in range(0, n, step):
        rows = q[r:r + step].double()
        m = rows.shape[0]
        x = rows.view(m, hkv, group, d).permute(1, 2, 0, 3).reshape(hkv, group * m, d)
        p = torch.bmm(x, kt).mul_(d ** -0.5).view(hkv, group, m, t)
        if causal:
            limit = torch.arange(first + r, first + r + m, device="cuda")
            p.masked_fill_(torch.arange(t, device="cuda")[None] > limit[:, None], -math.inf)
        total = torch.logsumexp(p, -1)
        p = (p - total[..., None].nan_to_num(neginf=0.0)).exp_().view(hkv, group * m, t)
        out[r:r + m] = torch.bmm(p, vt).view(hkv, group, m, d).permute(2, 0, 1, 3).reshape(m, hq, d)
        lse[r:r + m] = total.permute(2, 0, 1).reshape(m, hq)
    return out, lse


def _exact_cache_rows(s, name, b, n):
    pages = s["table"][b, :-(-n // s["page"])].long()
    x = s[name + "_cache"][pages].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][pages].double()[..., None]
    return x.reshape(-1, *x.shape[2:])[:n]


def _exact_append(s, new, total):
    t = s["q"].shape[0]
    where = [(b, total[b] - n + i) for b, n in enumerate(new) for i in range(n)]
    table = s["table"].cpu()
    slots = torch.tensor([int(table[b, p // s["page"]]) * s["page"] + p % s["page"] for b, p in where], device="cuda")
    angles = s["rotary"].double()[torch.tensor([p for _, p in where], device="cuda")]
    half = angles.shape[1] // 2
    turn = torch.complex(angles[:, :half], angles[:, half:])[:, None]

    def rotated(x):
        x = x.double().clone()
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["interleaved"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
        x[..., a], x[..., b] = z.real, z.imag
        return x

    def held(cache, rows):
        whole = torch.zeros(cache.shape[0] * cache.shape[1], *rows.shape[1:], dtype=torch.float64, device="cuda")
        whole[slots] = rows
        return whole.view(cache.shape)

    q, rows = rotated(s["q"]), [rotated(s["k"]), s["v"].double()]
    assert q.shape[0] == t
    if s["k_scale"] is None:
        return (q, *(held(s["k_cache"], x) for x in rows))
    scales = [x.abs().amax(-1).clamp(min=1e-12) / _FP8_MAX for x in rows]
    return (q, *(held(s["k_cache"], x / y[..., None]) for x, y in zip(rows, scales)), *(held(s["k_scale"], y) for y in scales))


def exact(case, seed):
    s = prepare(case, seed)
    new, total = _lengths(case)
    if case["kind"] == "append":
        return _exact_append(s, new, total)
    parts, at_q, at_k = [], 0, 0
    for b, (n, t) in enumerate(zip(new, total)):
        if case["kind"] == "decode":
            k, v = _exact_cache_rows(s, "k", b, t), _exact_cache_rows(s, "v", b, t)
        else:
            k, v = s["k"][at_k:at_k + t], s["v"][at_k:at_k + t]
            at_k += t
        parts.append(_exact_rows(s["q"][at_q:at_q + n], k, v, t - n, case["kind"] == "prompt" and case["causal"]))
        at_q += n
    return torch.cat([o for o, _ in parts]), torch.cat([x for _, x in parts])
