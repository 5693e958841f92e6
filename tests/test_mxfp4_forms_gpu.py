"""Every form of the MXFP4 products (bf16 and fp16 results, with and without bias, gated, of groups) with every kernel, scales read where they lie and arranged.

The kernel that a size gets is pinned (for the 256 compute units of a whole MI355X), so that a rule that moves takes no kernel out of the tests.
Operands and tolerances are those of test_mxfp4_gpu.py.
"""
import pytest
import torch

import mslk_amd
from oracle import mxfp4_oracle as O
from tests.helpers import mxfp4_kernel
from tests.test_mxfp4_gpu import BF16, DEV, F16, F32, gpu, grouped_oracle, operand, rng, same_bits, within

pytestmark = pytest.mark.gpu

# m, columns, k (gated: half as many of each), the kernel; several pairs of steps for each wave, and K that ends inside a step.
FORMS = [
    (5, 3000, 2912, "mx_stream<8,waves=8>"), (12, 3002, 288, "mx_stream<16,waves=8>"), (20, 3000, 2912, "mx_stream<32,waves=8>"),
    (40, 2000, 4736, "mx_tiles<32,32,waves=1x1x4>"), (40, 1998, 2080, "arrange_scales + mx_tiles<32,32,waves=1x1x4>"),
    (100, 2600, 4480, "mx_tiles<32,64,waves=1x1x4>"), (100, 2602, 2080, "arrange_scales + mx_tiles<32,64,waves=1x1x4>"),
    (128, 8192, 2176, "mx_tiles<64,64,waves=1x1x4>"), (97, 8190, 2080, "arrange_scales + mx_tiles<64,64,waves=1x1x4>"),
    (256, 8192, 2432, "mx_tiles<64,64,waves=1x1x2>"), (250, 8190, 2080, "arrange_scales + mx_tiles<64,64,waves=1x1x2>"), (16, 28672, 4096, "mx_tiles<64,64,waves=1x1x2>"),
    (500, 8192, 2048, "mx_tiles<128,128,waves=2x2x1>"), (500, 8190, 1568, "arrange_scales + mx_tiles<128,128,waves=2x2x1>"),
    (1100, 8192, 1024, "mx_walk"), (1100, 8190, 1568, "arrange_scales + mx_walk"), (1024, 10240, 800, "arrange_scales + mx_walk"),
]


def kernel(*args, **options):
    """Without its counts."""
    return mxfp4_kernel(*args, **options).split(" tiles=")[0].split(" workgroups=")[0]


def check_gated(got, xq, wq, xs, ws, what):
    want, (gate, _, _, _) = O.gated(xq, wq, xs, ws)
    within(got, want, (2.0 ** -20 + gate.abs() * 2.0 ** -22) * want.abs() + 1e-37, what)


@pytest.mark.parametrize("m,n,k,name", FORMS)
def test_dense(m, n, k, name):
    assert kernel(m, n, k) == name
    g = rng(m + n + k)
    xq, xs = operand(m, k, g)
    wq, ws = operand(n, k, g)
    want, size = O.product(xq, wq, xs, ws)
    assert size.max() < 1 << 20
    args = gpu(xq, wq, xs, ws)
    for dtype in (BF16, F16):
        same_bits(mslk_amd.mxfp4_mm(*args, out_dtype=dtype), want, f"{dtype}")
        for bias_dtype in (F32, BF16):
            bias = torch.randint(-64, 65, (n,), generator=g).to(bias_dtype)
            same_bits(mslk_amd.mxfp4_mm(*args, bias=bias.to(DEV), out_dtype=dtype), want + bias.double(), f"bias {bias_dtype}, {dtype}")


@pytest.mark.parametrize("m,n,k,name", FORMS)
def test_gated(m, n, k, name):
    assert kernel(m, n // 2, k, gated=True) == name
    g = rng(m + n + k + 1)
    xq, xs = operand(m, k, g)
    wq, ws = operand(n, k, g)
    ws -= 7
    for dtype in (BF16, F16):
        check_gated(mslk_amd.mxfp4_gated_mm(*gpu(xq, wq, xs, ws), out_dtype=dtype), xq, wq, xs, ws, f"{dtype}")


GROUP_FORMS = [
    ([3, 0, 130], 2000, 4480, "mx_tiles<64,64,waves=1x1x4> groups"), ([3, 0, 130], 2002, 2080, "arrange_scales + mx_tiles<64,64,waves=1x1x4> groups"),
    ([3, 0, 130], 4000, 2432, "mx_tiles<64,64,waves=1x1x2> groups"), ([3, 0, 130], 4002, 2080, "arrange_scales + mx_tiles<64,64,waves=1x1x2> groups"),
    ([20, 0, 9, 1], 8320, 2048, "mx_tiles<64,128,waves=2x2x1> groups"), ([100, 0, 33, 7], 8192, 1568, "arrange_scales + mx_tiles<64,128,waves=2x2x1> groups"),
    ([300, 1, 0, 256, 257, 2], 4096, 1024, "list_row_tiles + mx_walk groups"), ([300, 1, 0, 256, 257, 2], 4098, 1568, "arrange_scales with list_row_tiles + mx_walk groups"),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes,n,k,name", GROUP_FORMS)
def test_groups(sizes, n, k, name, gated, dtype):
    assert kernel(sum(sizes), n // 2 if gated else n, k, gated=gated, groups=len(sizes)) == name
    g = rng(n + k)
    xq, xs = operand(sum(sizes), k, g)
    wq, ws = operand((len(sizes), n), k, g)
    if gated:
        ws -= 7
    got = mslk_amd.mxfp4_grouped_mm(*gpu(xq, wq, xs, ws), torch.tensor(sizes, device=DEV), gated=gated, out_dtype=dtype)
    assert got.dtype == dtype
    if not gated:
        return same_bits(got, grouped_oracle(xq, wq, xs, ws, sizes, False))
    at = 0
    for e, rows in enumerate(sizes):
        if rows:
            check_gated(got[at:at + rows], xq[at:at + rows], wq[e], xs[at:at + rows], ws[e], f"group {e}")
        at += rows


# Products of so many steps that scales are arranged though they could be read where they lie: rows and columns from all over.
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("form", ["plain", "bias", "gated"])
def test_scales_arranged_for_a_large_product(form, dtype):
    m, n, k = 8200, 8192, 8192
    gated = form == "gated"
    assert kernel(m, n // 2 if gated else n, k, gated=gated) == "arrange_scales + mx_walk"
    gen = torch.Generator(DEV).manual_seed(3)
    byte = lambda low, high, *shape: torch.randint(low, high, shape, generator=gen, device=DEV, dtype=torch.uint8)  # noqa: E731
    xq, xs, wq, ws = byte(0, 256, m, k // 2), byte(126, 129, m, k // 32), byte(0, 256, n, k // 2), byte(126 - 7 * gated, 129 - 7 * gated, n, k // 32)
    rows = torch.cat([torch.arange(0, m, 97), torch.arange(m - 9, m)]).to(DEV)
    if gated:
        columns = torch.cat([torch.arange(0, n // 2, 61), torch.arange(n // 2 - 3, n // 2)]).to(DEV)
        both = torch.cat([columns, columns + n // 2])
        got = mslk_amd.mxfp4_gated_mm(xq, wq, xs, ws, out_dtype=dtype)[rows][:, columns]
        return check_gated(got, xq[rows].cpu(), wq[both].cpu(), xs[rows].cpu(), ws[both].cpu(), form)
    columns = torch.cat([torch.arange(0, n, 61), torch.arange(n - 3, n)]).to(DEV)
    bias = torch.randint(-64, 65, (n,), generator=gen, device=DEV).float() if form == "bias" else None
    got = mslk_amd.mxfp4_mm(xq, wq, xs, ws, bias=bias, out_dtype=dtype)[rows][:, columns]
    want, size = O.product(xq[rows], wq[columns], xs[rows], ws[columns], None if bias is None else bias[columns])
    assert size.max() < 1 << 20
    same_bits(got, want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("gated", [False, True])
def test_scales_arranged_for_large_products_of_groups(gated, dtype):
    sizes, n, k = [9000, 0, 7001, 500], 8192, 4096
    m = sum(sizes)
    assert kernel(m, n // 2 if gated else n, k, gated=gated, groups=4) == "arrange_scales with list_row_tiles + mx_walk groups"
    gen = torch.Generator(DEV).manual_seed(4)
    byte = lambda low, high, *shape: torch.randint(low, high, shape, generator=gen, device=DEV, dtype=torch.uint8)  # noqa: E731
    xq, xs, wq, ws = byte(0, 256, m, k // 2), byte(126, 129, m, k // 32), byte(0, 256, 4, n, k // 2), byte(126 - 7 * gated, 129 - 7 * gated, 4, n, k // 32)
    y = mslk_amd.mxfp4_grouped_mm(xq, wq, xs, ws, torch.tensor(sizes, device=DEV), gated=gated, out_dtype=dtype)
    at = 0
    for e, size in enumerate(sizes):
        if size == 0:
            continue
        rows = torch.cat([torch.arange(at, at + size, 97), torch.arange(at + size - 3, at + size)]).to(DEV)
        columns = torch.arange(0, n // 2 if gated else n, 61, device=DEV)
        of_w = torch.cat([columns, columns + n // 2]) if gated else columns
        got, args = y[rows][:, columns], (xq[rows].cpu(), wq[e][of_w].cpu(), xs[rows].cpu(), ws[e][of_w].cpu())
        at += size
        if gated:
            check_gated(got, *args, f"group {e}")
        else:
            same_bits(got, O.product(*args)[0], f"group {e}")


# Powers at both ends of their range: the instruction adds the scales' exponents, nothing overflows on the way.
SCALES = [0, 1, 60, 126, 127, 128, 200, 253, 254]


@pytest.mark.parametrize("m,n,k", [(9, 90, 96), (40, 300, 128), (520, 4000, 64), (520, 4000, 512), (1100, 8000, 544)])
def test_scales_at_both_ends(m, n, k):
    """One product per result, up to 36 times 2^254 and down to 2^-256: infinite, exact or 0 as its rounding is."""
    xq, wq = torch.zeros(m, k // 2, dtype=torch.uint8), torch.zeros(n, k // 2, dtype=torch.uint8)
    xs, ws = (torch.randint(0, 255, (r, k // 32), generator=rng(r), dtype=torch.uint8) for r in (m, n))
    xq[:, k // 2 - 3] = 7
    wq[:, k // 2 - 3] = torch.tensor([13, 3, 7, 1], dtype=torch.uint8)[torch.arange(n) % 4]
    xs[:, -1] = torch.tensor(SCALES, dtype=torch.uint8)[torch.arange(m) % 9]
    ws[:, -1] = torch.tensor(SCALES, dtype=torch.uint8)[torch.arange(n) // 4 % 9]
    same_bits(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws)), O.product(xq, wq, xs, ws)[0])


def test_views_of_the_torch_types():
    """Codes that begin inside 16 bytes and scales with a stride, as float4_e2m1fn_x2 and float8_e8m0fnu: both are copied."""
    g = rng(8)
    xq, xs = gpu(*operand(40, 1024, g))
    wq, ws = gpu(*operand(30, 1024, g))
    want = O.product(xq, wq, xs, ws)[0]

    def moved(t, by):
        flat = torch.zeros(t.numel() + by, dtype=torch.uint8, device=DEV)
        flat[by:] = t.flatten()
        return flat[by:].view(t.shape).view(torch.float4_e2m1fn_x2)

    strided = torch.zeros(30, 40, dtype=torch.uint8, device=DEV)
    strided[:, 3:35] = ws
    scales = strided.view(torch.float8_e8m0fnu)[:, 3:35]
    same_bits(mslk_amd.mxfp4_mm(moved(xq, 8), wq, xs, scales), want)
    same_bits(mslk_amd.mxfp4_grouped_mm(moved(xq, 8), moved(wq[None], 4), xs, scales[None], torch.tensor([40], device=DEV)), want)
    same_bits(mslk_amd.dequantize_mxfp4(moved(xq, 1), xs.view(torch.float8_e8m0fnu)), O.values(xq, xs))
