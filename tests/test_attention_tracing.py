"""append_kv writes its caches in place: with tensors that have no data, traced into a functional graph.  No GPU needed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mslk_amd


def arguments(fp8, empty):
    cache = mslk_amd.FP8_DTYPE if fp8 else torch.bfloat16
    pools = [empty(3, 16, 2, 64, dtype=cache) for _ in range(2)]
    scales = [empty(3, 16, 2) for _ in range(2)] if fp8 else [None, None]
    q, k, v = (empty(4, n, 64, dtype=torch.bfloat16) for n in (4, 2, 2))
    return q, k, v, *pools, empty(4, 2, dtype=torch.int32), empty(4, dtype=torch.int32), *scales


def append(q, k, v, k_cache, v_cache, table, lens, k_scale=None, v_scale=None):
    return torch.ops.mslk.append_kv(q, k, v, k_cache, v_cache, table, lens, None, None, False, k_scale, v_scale)


@pytest.mark.parametrize("fp8", [False, True])
def test_versions_of_the_caches_move(fp8):
    with FakeTensorMode():
        args = arguments(fp8, lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda"))
        before = [None if t is None else t._version for t in args]
        out = append(*args)
        assert out.shape == (4, 4, 64) and out.dtype == torch.bfloat16
        for i, (t, was) in enumerate(zip(args, before)):
            if t is not None:
                assert (t._version > was) == (i in (3, 4, 7, 8)), i


@pytest.mark.parametrize("fp8", [False, True])
def test_exporting_keeps_the_writes(fp8):
    """Functionalized, the program hands back the caches as the operator leaves them."""
    class Step(torch.nn.Module):
        def forward(self, *args):
            return append(*args)

    with FakeTensorMode():
        args = arguments(fp8, lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda"))
        args = tuple(t for t in args if t is not None)
        program = torch.export.export(Step(), args).run_decompositions()
    assert len(program.graph_signature.user_inputs_to_mutate) == (4 if fp8 else 2), program
