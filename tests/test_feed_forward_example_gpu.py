"""examples/serve_feed_forward.py runs: a shared block and routed experts in one captured graph, replays equal to eager steps."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("options", [[], ["--hidden", "512", "--width", "1056", "--expert-width", "160", "--experts", "5", "--top", "2", "--tokens", "7"],
                                     ["--hidden", "1024", "--tokens", "1"], ["--tokens", "700", "--steps", "3"]])
def test_replays_equal_eager_steps(options):
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "serve_feed_forward.py")
    spec = importlib.util.spec_from_file_location("serve_feed_forward", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    same, error = example.main(["--steps", "4", *options])
    assert same
    # A code is off by at most a fourth of its value and a twelfth of the block's largest one, so every quantized operand keeps a
    # cosine above 0.9 with its values and two products in a row keep some of it: a result of other rows or weights has none.
    assert error < 1.0
