"""Both parts of examples/serve_feed_forward.py, one at a time, against the same layer in 64 bits from its codes and scales.

What is allowed is 2^-6 of the result's norm.  Results that are rounded are off by 2^-9.  A hidden value whose fp32 sum lands on the other side of a rounding to
bf16 (less than one in 2^7: sums are off by 2^-16 of their size, a step is 2^-8) gets another code if a boundary of codes lies between the two, which of
the 2^7 numbers of a binade three or fewer have: less than one code in 2^12 differs, by at most a third of its value, 2^-6 / 3 of the norm.  Rows of another
token or expert, or a part that is missing, differ by about the norm itself.
"""
import importlib.util
import os

import pytest
import torch

from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "serve_feed_forward.py")
    spec = importlib.util.spec_from_file_location("serve_feed_forward", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def block(x, up, down):
    xq, xs = O.quantize(x)
    hq, hs = O.quantize(O.gated(xq, up[0], xs, up[1])[0].bfloat16())
    return O.product(hq, down[0], hs, down[1])[0]


def expected(layer, x, part):
    w = {name: tuple(t.cpu() for t in pair) for name, pair in layer.weights.items()}
    if part == "shared":
        return block(x.cpu(), w["up"], w["down"])
    scores, chosen = torch.softmax((x @ layer.router.t()).float(), -1).topk(layer.top)
    scores, chosen, x = (scores / scores.sum(-1, keepdim=True)).double().cpu(), chosen.cpu(), x.cpu()
    y = torch.zeros(x.shape, dtype=torch.float64)
    for e in range(layer.experts):
        token, choice = (chosen == e).nonzero(as_tuple=True)
        if len(token):
            y[token] += scores[token, choice, None] * block(x[token], *(tuple(t[e] for t in w[name]) for name in ("expert_up", "expert_down")))
    return y


@pytest.mark.parametrize("part,other", [("shared", "expert_down"), ("routed", "down")])
@pytest.mark.parametrize("hidden,width,expert_width,experts,top,tokens", [(512, 1056, 160, 5, 2, 7), (1024, 2048, 544, 8, 3, 150), (512, 512, 288, 4, 1, 1)])
def test_part(part, other, hidden, width, expert_width, experts, top, tokens):
    torch.manual_seed(hidden + tokens)
    layer = example().FeedForward(hidden, width, expert_width, experts, top)
    layer.weights[other][0].zero_()   # the other part adds nothing
    x = torch.randn(tokens, hidden, device="cuda").bfloat16()
    got, want = layer(x).double().cpu(), expected(layer, x, part)
    assert ((got - want).norm() <= 2.0 ** -6 * want.norm()), ((got - want).norm() / want.norm())
