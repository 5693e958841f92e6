"""Attention of a served decoder layer: new keys and values into a paged cache, one new token per sequence over that cache, and
whole prompts packed one after the other.

The operators are `torch.ops.mslk.append_kv`, `attention_decode` and `attention_prompt` (GPU kernels only, native:
csrc/torch_ops.cpp; csrc/append_kv.hip, attention_decode.hip, attention_prompt.hip); the functions below are their Python form.
They have no counterpart in the reference's FP8 path: they are what a program puts between its FP8 projections.

A cache is two tensors [pages, page_size, kv_heads, channels], in the type of the queries or in float8_e4m3fn with one fp32 scale
per row (`k_scale`, `v_scale` [pages, page_size, kv_heads]).  Strides are free as long as channels are contiguous, so a
pool [pages, kv_heads, page_size, channels] is passed as `pool.transpose(1, 2)`; scales kept by head like that, [pages, kv_heads,
page_size], are read with fewer bytes, because a head's lie side by side.  `page_table` [sequences, width] (int32) names the
pages of each sequence in order, `kv_lens` [sequences] (int32) says how many keys it has; both are read on the GPU only, so a
captured graph follows them.  Nothing here is differentiable.

Scores, softmax statistics and sums are fp32.  `attention_decode` keeps 16 bits or more of each softmax weight, so that its output is off
by its one rounding; `attention_prompt` rounds the weights to the type of the queries, which adds about as much again (relative to 64
bits 0.002 instead of 0.0016 in bf16, 0.00028 instead of 0.0002 in fp16).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

_library = torch.library.Library("mslk", "FRAGMENT")


def _fake_append_kv(q, k, v, k_cache, v_cache, page_table, kv_lens, cu_seqlens=None, rotary=None, interleaved=False, k_scale=None,
                    v_scale=None):
    for t in (k_cache, v_cache, k_scale, v_scale):   # written, as far as autograd is concerned
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _fake_attention(q, *args, **kwargs):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)


_OPS = {
    "append_kv": ("(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor kv_lens, "
                  "Tensor? cu_seqlens=None, Tensor? rotary=None, bool interleaved=False, Tensor(c!)? k_scale=None, "
                  "Tensor(d!)? v_scale=None) -> Tensor", _fake_append_kv),
    "attention_decode": ("(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor kv_lens, Tensor? k_scale=None, "
                         "Tensor? v_scale=None, float? scale=None) -> (Tensor, Tensor)", _fake_attention),
    "attention_prompt": ("(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens, Tensor? cu_seqlens_k=None, bool causal=True, "
                         "float? scale=None) -> (Tensor, Tensor)", _fake_attention),
}
for _name, (_schema, _fake) in _OPS.items():
    if not hasattr(torch.ops.mslk, _name):
        _library.define(_name + _schema)
        torch.library.register_fake(f"mslk::{_name}", _fake, lib=_library)
    # Outside of autograd: without a derivative its fallback would make the results part of the graph of any input that requires a
    # gradient.  (Calling under no_grad() instead costs 1.5 us, a quarter of a small call.)
    _library.impl(_name, torch.library.fallthrough_kernel, "Autograd")


def _check_gpu(name: str, q: torch.Tensor) -> None:
    if not q.is_cuda:
        raise RuntimeError(f"mslk_amd.{name}: inputs must be GPU tensors (no CPU implementation)")


def append_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, kv_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
              rotary: Optional[torch.Tensor] = None, interleaved: bool = False, k_scale: Optional[torch.Tensor] = None,
              v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates q [T, Hq, D] and k [T, Hkv, D] by their positions, writes k and v into the cache, returns the rotated q.

    `cu_seqlens` [sequences + 1] (int32) says where the new tokens of each sequence begin; without it there is one per sequence.
    They take the last positions of the sequence's `kv_lens` keys, which count them already.  `rotary` [positions, R] (fp32, R even,
    at most D) holds cosines and then sines; it turns channels i and i + R / 2 (`interleaved`: 2 i and 2 i + 1) into
    (a cos - b sin, b cos + a sin).  q, k and v may be views of one projection's output.

    Tokens of no sequence and positions below zero are padding: a query of zeros, nothing stored.  A position beyond `rotary` or
    without a page stores nothing and gives a query of NaN."""
    _check_gpu("append_kv", q)
    return torch.ops.mslk.append_kv(q, k, v, k_cache, v_cache, page_table, kv_lens, cu_seqlens, rotary, interleaved, k_scale, v_scale)


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of q [sequences, Hq, D], one token per sequence, over the first `kv_lens` keys of each sequence's pages.

    Returns out [sequences, Hq, D] and, with `return_lse`, log sum exp of the scaled scores [sequences, Hq] (fp32).  `scale` is
    1 / sqrt(D) unless given (positive, at most 2e38).  A sequence without keys gives zeros and -inf; one whose keys lack a page gives NaN."""
    _check_gpu("attention_decode", q)
    out, lse = torch.ops.mslk.attention_decode(q, k_cache, v_cache, page_table, kv_lens, k_scale, v_scale, scale)
    return (out, lse) if return_lse else out


def attention_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = True, scale: Optional[float] = None,
                     return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of packed prompts: q [T, Hq, D] over k, v [S, Hkv, D], sequence b at cu_seqlens[b] ... cu_seqlens[b + 1] - 1
    (keys: `cu_seqlens_k`, if they are not as many as the queries).

    `causal`: the last query of a sequence sees its last key, each one before it a key less.  Queries that see nothing, and tokens
    of no sequence, give zeros and -inf.  Returns as `attention_decode`."""
    _check_gpu("attention_prompt", q)
    out, lse = torch.ops.mslk.attention_prompt(q, k, v, cu_seqlens, cu_seqlens_k, causal, scale)
    return (out, lse) if return_lse else out
