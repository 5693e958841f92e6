"""MXFP4 products of more rows than one dimension of a launch holds (2^32 work-items), up to 2^31 - 1: rows from all over, and the last ones."""
import pytest
import torch

import mslk_amd
from oracle import mxfp4_oracle as O
from tests.test_mxfp4_gpu import DEV, same_bits

pytestmark = pytest.mark.gpu
K = 32


def operand(rows, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (rows, K // 2), generator=gen, device=DEV, dtype=torch.uint8)
    return codes, torch.randint(126, 129, (rows, 1), generator=gen, device=DEV, dtype=torch.uint8)


def some(size):
    at = torch.cat([torch.arange(200), torch.randint(0, size, (2000,), generator=torch.Generator().manual_seed(1)), torch.arange(size - 200, size)])
    return at.clamp(0, size - 1).unique().to(DEV)


@pytest.fixture(autouse=True)
def memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m,n", [(2 ** 29 + 77, 3), (2, 2 ** 29 + 77), (2 ** 31 - 1, 1), (1, 2 ** 31 - 1)])
def test_rows_beyond_a_launch(m, n):
    (xq, xs), (wq, ws) = operand(m, 1), operand(n, 2)
    y = mslk_amd.mxfp4_mm(xq, wq, xs, ws)
    rows, columns = some(m), some(n)
    same_bits(y[rows][:, columns], O.product(xq[rows], wq[columns], xs[rows], ws[columns])[0])


@pytest.mark.parametrize("sizes", [[5, 2 ** 30 + 100, 0, 95], [2 ** 31 - 1]], ids=["four", "one"])
def test_rows_of_experts_beyond_a_launch(sizes):
    """Row tiles of 64 in more than 2^24 workgroups."""
    m, n, groups = sum(sizes), 2, len(sizes)
    (xq, xs), (wq, ws) = operand(m, 3), operand(groups * n, 4)
    wq, ws = wq.view(groups, n, -1), ws.view(groups, n, -1)
    y = mslk_amd.mxfp4_grouped_mm(xq, wq, xs, ws, torch.tensor(sizes, device=DEV))
    rows = some(m)
    got = y[rows]
    group = torch.bucketize(rows.cpu(), torch.tensor(sizes).cumsum(0), right=True)
    for g in group.unique().tolist():
        at = (group == g).nonzero().flatten()
        picked = rows[at.to(DEV)]
        same_bits(got[at.to(DEV)], O.product(xq[picked], wq[g], xs[picked], ws[g])[0], f"group {g}")
