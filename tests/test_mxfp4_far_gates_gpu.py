"""Gates from -85 to -192 beside partners up to 2^127: silu(gate) passes the smallest normal number there, its product with the partner does not.

Both factors are exact sums (whole and half units; one product), so what is allowed is what test_mxfp4_gpu.py allows for the exponential, 2^-20 + |gate| 2^-22 of
the result, and 2^-140 for a partner times exp(gate) below the normal numbers: off by 2^-150, times a gate below 2^8.
"""
import pytest
import torch

import mslk_amd
from oracle import mxfp4_oracle as O
from tests.test_mxfp4_gpu import BF16, DEV, F16, gpu, within

pytestmark = pytest.mark.gpu
HALVES = [12, 8, 6, 4, 3, 2, 1]   # what the codes 7 ... 1 stand for, in halves
FACTORS = [2, 1, 10]              # codes of 1, 0.5, -1: the three kinds of rows of X


def weights(n, k):
    """Gate rows -85, -85.5, ... in block 0, partners 1.5 2^p in block 1; p so that the results are near 1 while the type of p has room."""
    codes, scales = torch.zeros(2 * n, k, dtype=torch.uint8), torch.full((2 * n, k // 32), 127, dtype=torch.uint8)
    for c in range(n):
        halves = 170 + c % 215
        gate, at = halves / 2, 0
        for code, size in zip(range(7, 0, -1), HALVES):
            while halves >= size:
                codes[c, at] = 8 | code
                halves, at = halves - size, at + 1
        codes[n + c, 32] = 3 | (c // 215 % 2) << 3
        scales[n + c, 1] = 127 + min(127, round(gate * 1.4427 - 7) + c % 17 - 8)
    return codes[:, ::2] | (codes[:, 1::2] << 4), scales


def rows(m, k):
    codes = torch.randint(0, 256, (3, k // 2), generator=torch.Generator().manual_seed(k), dtype=torch.uint8)
    codes[:, :16], codes[:, 16] = 0x22, torch.tensor(FACTORS, dtype=torch.uint8)
    scales = torch.full((3, k // 32), 127, dtype=torch.uint8)
    kind = torch.arange(m) % 3
    return codes, scales, kind


def check(got, codes, scales, kind, wq, ws):
    want, (gate, up, _, _) = O.gated(codes, wq, scales, ws)
    assert gate.max() == -85 and gate.min() <= -192 or gate.shape[1] < 215
    want, gate = want[kind], gate[kind]
    assert (want.abs() > 2.0 ** -24).any() and torch.isfinite(want).all()
    within(got, want, (2.0 ** -20 + gate.abs() * 2.0 ** -22) * want.abs() + 2.0 ** -140)


# streamed; 32 x 32, 32 x 64, 64 x 64 tiles of four and of two waves, 128 x 128 ones; 256-column ones, whole and not
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(2, 215, 96), (20, 430, 4128), (40, 300, 128), (40, 3000, 128), (40, 4300, 128), (40, 9000, 128), (520, 4000, 64), (520, 4000, 512),
                                   (1024, 4096, 544), (1100, 4001, 512)])
def test_far_gates(m, n, k, dtype):
    codes, scales, kind = rows(m, k)
    wq, ws = weights(n, k)
    check(mslk_amd.mxfp4_gated_mm(*gpu(codes[kind], wq, scales[kind], ws), out_dtype=dtype), codes, scales, kind, wq, ws)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,n,k", [([5, 0, 40], 300, 128), ([300, 1, 0, 256, 257, 2], 1000, 160), ([300, 100], 3000, 544)])
def test_far_gates_of_experts(sizes, n, k, dtype):
    codes, scales, kind = rows(sum(sizes), k)
    wq, ws = weights(n, k)
    stacked = [t.expand(len(sizes), *t.shape).contiguous() for t in (wq, ws)]
    got = mslk_amd.mxfp4_grouped_mm(*gpu(codes[kind], stacked[0], scales[kind], stacked[1]), torch.tensor(sizes, device=DEV), gated=True, out_dtype=dtype)
    check(got, codes, scales, kind, wq, ws)


def test_gates_of_minus_infinity_and_nan():
    """A gate that is NaN, or whose fp32 sum is infinite, is what gate * sigmoid(gate) makes of it: NaN."""
    codes, scales, kind = rows(3, 64)
    wq, ws = weights(4, 64)
    ws[1, 0] = 255
    wq[2], ws[2] = 0xFF, 254   # -6 2^127, and more of it
    got = mslk_amd.mxfp4_gated_mm(*gpu(codes, wq, scales, ws)).cpu()
    assert torch.isnan(got[:, 1:3]).all() and torch.isfinite(got[:, [0, 3]]).all()
