"""examples/serve_attention.py: projections, cache and attention together, steps against one pass over the whole sequences."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("options", [[], ["--fp8-cache"], ["--head-dim", "80", "--heads", "12", "--kv-heads", "4", "--page-size", "7"]])
def test_steps_agree_with_one_pass(options):
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "serve_attention.py")
    spec = importlib.util.spec_from_file_location("serve_attention", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # Both sides round the attention's output to 16 bits (2^-9 relative, independent) and then to e4m3, where a difference moves about
    # one code in ten by 2^-4 of its size: 2^-4 / sqrt(10) = 0.02; two more sources of this size with an e4m3 cache's own read-back.
    assert example.main(["--steps", "5", "--hidden", "1024", *options]) < 0.05
