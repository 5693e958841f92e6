"""The attention of a decoder layer as a server runs it: prompts packed one after the other, then one token per sequence and step.

    python examples/serve_attention.py [--hidden 2048] [--heads 16] [--kv-heads 8] [--head-dim 128] [--steps 32] [--fp8-cache]

FP8 projections (quantize_fp8_row, f8f8bf16_rowwise) around append_kv, attention_prompt and attention_decode, with random weights and
inputs.  The steps run as a captured graph that counts the keys itself.  At the end the outputs of the steps are compared with those of
one pass over the whole sequences.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mslk_amd  # noqa: E402


class PagedCache:
    """Keys and values of up to `sequences` sequences of `longest` tokens, in pages handed out in any order."""

    def __init__(self, sequences, longest, kv_heads, head_dim, page_size, fp8):
        width = -(-longest // page_size)
        shape = (sequences * width, page_size, kv_heads)
        dtype = mslk_amd.FP8_DTYPE if fp8 else torch.bfloat16
        self.k, self.v = (torch.zeros(*shape, head_dim, dtype=dtype, device="cuda") for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(shape, device="cuda") if fp8 else None for _ in range(2))
        self.table = torch.randperm(sequences * width).view(sequences, width).to(torch.int32).cuda()
        self.lens = torch.zeros(sequences, dtype=torch.int32, device="cuda")

    def rows(self, lens):
        """The first lens[b] keys and values of each sequence, packed: what a prompt attends to, cached parts included."""
        page = self.k.shape[1]
        at = torch.cat([self.table[b].long()[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page
                        for b, n in enumerate(lens)])
        packed = [x.view(-1, *x.shape[2:]).view(torch.uint8 if x.element_size() == 1 else x.dtype)[at].view(x.dtype) for x in (self.k, self.v)]
        if self.k_scale is None:
            return packed
        scales = [x.view(-1, x.shape[2])[at] for x in (self.k_scale, self.v_scale)]
        return [(x.float() * s[..., None]).bfloat16() for x, s in zip(packed, scales)]


class Attention:
    def __init__(self, hidden, heads, kv_heads, head_dim, positions):
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        weights = [torch.randn(n, k, device="cuda").bfloat16() / k ** 0.5
                   for n, k in (((heads + 2 * kv_heads) * head_dim, hidden), (hidden, heads * head_dim))]
        self.qkv, self.out = (mslk_amd.quantize_fp8_row(w) for w in weights)
        angles = torch.arange(positions, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, head_dim, 2, device="cuda") / head_dim)
        self.rotary = torch.cat([angles.cos(), angles.sin()], 1)

    @staticmethod
    def linear(x, weight):
        xq, scale = mslk_amd.quantize_fp8_row(x)
        return torch.ops.mslk.f8f8bf16_rowwise(xq, weight[0], scale, weight[1])

    def __call__(self, x, cache, cu_seqlens=None, lens=None):
        """x: packed new tokens, one per sequence without `cu_seqlens`; cache.lens counts them.  `lens`: cache.lens on the host."""
        qkv = self.linear(x, self.qkv).view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
        q = mslk_amd.append_kv(q, k, v, cache.k, cache.v, cache.table, cache.lens, cu_seqlens, self.rotary, k_scale=cache.k_scale,
                               v_scale=cache.v_scale)
        if cu_seqlens is None:
            o = mslk_amd.attention_decode(q, cache.k, cache.v, cache.table, cache.lens, cache.k_scale, cache.v_scale)
        else:
            o = mslk_amd.attention_prompt(q, *cache.rows(lens), cu_seqlens, offsets(lens))
        return self.linear(o.flatten(1), self.out)


def offsets(lens):
    return torch.tensor([0, *lens], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("--hidden", 2048), ("--heads", 16), ("--kv-heads", 8), ("--head-dim", 128), ("--page-size", 16), ("--steps", 32)):
        parser.add_argument(name, type=int, default=value)
    parser.add_argument("--fp8-cache", action="store_true")
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    prompts = [700, 33, 1, 256, 129]
    longest = max(prompts) + args.steps
    layer = Attention(args.hidden, args.heads, args.kv_heads, args.head_dim, longest)
    new_cache = lambda: PagedCache(len(prompts), longest, args.kv_heads, args.head_dim, args.page_size, args.fp8_cache)  # noqa: E731
    tokens = [torch.randn(n + args.steps, args.hidden, device="cuda").bfloat16() for n in prompts]

    # The prompts in two passes: the first half of each, then the rest, which continues what is in the cache.
    cache = new_cache()
    halves = [n // 2 for n in prompts]
    for begin, end in (([0] * len(prompts), halves), (halves, prompts)):
        cache.lens.copy_(torch.tensor(end))
        layer(torch.cat([t[a:b] for t, a, b in zip(tokens, begin, end)]), cache, offsets([b - a for a, b in zip(begin, end)]), end)

    # The steps.
    x = torch.empty(len(prompts), args.hidden, dtype=torch.bfloat16, device="cuda")

    def step():
        cache.lens.add_(1)
        return layer(x, cache)

    stepped = []
    graph = None
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(args.steps):
        x.copy_(torch.stack([t[n + i] for t, n in zip(tokens, prompts)]))
        if graph is None and i > 0:   # (the first step has loaded every kernel)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured = step()
        start.record()
        if graph is None:
            out = step()
        else:
            graph.replay()
            out = captured
        stop.record()
        stepped.append(out.clone())
    torch.cuda.synchronize()
    us = start.elapsed_time(stop) * 1e3

    # Everything once more in one pass.
    whole = new_cache()
    lens = [n + args.steps for n in prompts]
    whole.lens.copy_(torch.tensor(lens))
    want = layer(torch.cat(tokens), whole, offsets(lens), lens)
    want = torch.stack([o[n:] for o, n in zip(want.split(lens), prompts)], 1).float()   # [steps, sequences, hidden]
    error = ((torch.stack(stepped).float() - want).norm() / want.norm()).item()
    print(f"{len(prompts)} sequences, {sum(prompts)} prompt tokens, {args.steps} steps, the last one in {us:.0f} us; "
          f"steps against one pass over the whole sequences: relative error {error:.4f}")
    return error


if __name__ == "__main__":
    # e4m3 rounds to 1 part in 16; what differs are roundings of 16-bit rows before them, so most codes are the same
    sys.exit(0 if main() < 0.05 else 1)
