"""The feed-forward half of a decoder layer as a server runs it, in MXFP4: a gated block that every token takes, and routed experts.

    python examples/serve_feed_forward.py [--hidden 2048] [--width 4096] [--expert-width 1024] [--experts 32] [--top 4] [--tokens 64]

Weights are quantized once (quantize_mxfp4), activations in front of each product; mxfp4_gated_mm and mxfp4_mm make the block that all
tokens share, mxfp4_grouped_mm the experts: a token's codes are copied once per expert that it goes to, in the order of the experts, whose
row counts stay on the GPU.  One step is a captured graph.  With random weights and inputs; at the end the result is compared with that of
the weights and activations in bf16.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mslk_amd  # noqa: E402


class FeedForward:
    def __init__(self, hidden, width, expert_width, experts, top):
        new = lambda *shape: torch.randn(*shape, device="cuda").bfloat16() / shape[-1] ** 0.5  # noqa: E731
        self.router = new(experts, hidden)
        self.plain = {"up": new(2 * width, hidden), "down": new(hidden, width),   # "up": gate rows, then those of its partner
                      "expert_up": new(experts, 2 * expert_width, hidden), "expert_down": new(experts, hidden, expert_width)}
        self.weights = {name: mslk_amd.quantize_mxfp4(w) for name, w in self.plain.items()}
        self.experts, self.top = experts, top

    def route(self, x):
        """For each of the tokens' choices, in the order of experts: its token; where a token's choices are; their weights; rows per expert."""
        scores, chosen = torch.softmax((x @ self.router.t()).float(), -1).topk(self.top)
        order = chosen.flatten().argsort(stable=True)
        place = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=x.device))
        counts = (chosen.flatten()[:, None] == torch.arange(self.experts, device=x.device)).sum(0)
        return order // self.top, place, scores / scores.sum(-1, keepdim=True), counts

    def __call__(self, x):
        (xq, xs), w = mslk_amd.quantize_mxfp4(x), self.weights
        hq, hs = mslk_amd.quantize_mxfp4(mslk_amd.mxfp4_gated_mm(xq, w["up"][0], xs, w["up"][1]))
        shared = mslk_amd.mxfp4_mm(hq, w["down"][0], hs, w["down"][1])
        token, place, scores, counts = self.route(x)
        h = mslk_amd.mxfp4_grouped_mm(xq[token], w["expert_up"][0], xs[token], w["expert_up"][1], counts, gated=True)
        hq, hs = mslk_amd.quantize_mxfp4(h)
        y = mslk_amd.mxfp4_grouped_mm(hq, w["expert_down"][0], hs, w["expert_down"][1], counts)
        routed = (y[place].view(*scores.shape, -1).float() * scores[..., None]).sum(1)
        return (shared.float() + routed).bfloat16()

    def in_bf16(self, x):
        def block(x, up, down):
            gate, other = (x @ up.t()).float().chunk(2, -1)
            return (torch.nn.functional.silu(gate) * other).bfloat16() @ down.t()

        token, place, scores, counts = self.route(x)
        parts = x[token].split(counts.tolist())
        y = torch.cat([block(part, self.plain["expert_up"][e], self.plain["expert_down"][e]) for e, part in enumerate(parts)])
        routed = (y[place].view(*scores.shape, -1).float() * scores[..., None]).sum(1)
        return (block(x, self.plain["up"], self.plain["down"]).float() + routed).bfloat16()


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("--hidden", 2048), ("--width", 4096), ("--expert-width", 1024), ("--experts", 32), ("--top", 4), ("--tokens", 64), ("--steps", 8)):
        parser.add_argument(name, type=int, default=value)
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    layer = FeedForward(args.hidden, args.width, args.expert_width, args.experts, args.top)
    x = torch.empty(args.tokens, args.hidden, dtype=torch.bfloat16, device="cuda").normal_()
    layer(x)   # (loads every kernel)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    same = True
    for _ in range(args.steps):
        x.normal_()
        start.record()
        graph.replay()
        stop.record()
        same &= torch.equal(out, layer(x))
    torch.cuda.synchronize()
    want = layer.in_bf16(x).float()
    error = ((out.float() - want).norm() / want.norm()).item()
    print(f"{args.tokens} tokens, {args.experts} experts, {args.top} of them per token, a step in {start.elapsed_time(stop) * 1e3:.0f} us; replayed steps "
          f"{'equal' if same else 'DIFFER FROM'} eager ones; against bf16: relative error {error:.3f}")
    return same, error


if __name__ == "__main__":
    sys.exit(0 if main()[0] else 1)
