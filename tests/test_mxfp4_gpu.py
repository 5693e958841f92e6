"""MXFP4 operators against their definition in 64 bits (oracle/mxfp4_oracle.py).

Two kinds of operands.  "Whole": scales of 2^-1, 1, 2 and any codes, so that every product is a multiple of 1/16 and sums below 2^20
are exact in fp32 in any order: results have to equal the rounded exact ones bit for bit.  "Wide": scales over many powers of two; a sum
of K terms passes K / 64 additions to an accumulator and at most 64 inside an instruction, each off by at most 2^-23 of at most
A = sum |x w|, so |y - exact| <= half a step of the output type + (K / 64 + 64) 2^-23 A.
"""
import pytest
import torch

import mslk_amd
from mslk_amd import _lib
from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rng(seed):
    return torch.Generator().manual_seed(seed)


def operand(rows, k, g, low=126, high=128):
    """Codes and scales (bytes from `low` to `high`) of rows [*rows, k]."""
    rows = rows if isinstance(rows, tuple) else (rows,)
    codes = torch.randint(0, 256, (*rows, k // 2), generator=g, dtype=torch.uint8)
    return codes, torch.randint(low, high + 1, (*rows, k // 32), generator=g, dtype=torch.uint8)


def gpu(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


def same_bits(got, want, what=""):
    """`want` in 64 bits, rounded once (NaN where it is)."""
    want = want.to(got.dtype)
    got = got.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    bad = (got != want) & ~nan
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} differ, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} instead of {want[bad][0]}"


def within(got, want, allowed, what=""):
    """Half a step of the output type and `allowed` more, for every element."""
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * eps   # half a step below the normal numbers
    off = (got.cpu().double() - want).abs() - ((want.abs() + allowed) * eps + allowed + tiny)
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} elements off by up to {off.max():.3g} more than allowed"


# ---------------------------------------------------------------------------------------------------------------------
# quantizer
# ---------------------------------------------------------------------------------------------------------------------
def check_quantized(a):
    """`a` may live anywhere and have any strides."""
    codes, scales = mslk_amd.quantize_mxfp4(a)
    want_codes, want_scales = O.quantize(a.cpu())
    assert codes.dtype == scales.dtype == torch.uint8
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu(), want_codes)
    return codes, scales


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 32), (1, 4096), (3, 96), (257, 2880), (0, 64), (5, 0), (64,), (2, 3, 160), (513, 4128)])
def test_quantize_rows(shape, dtype):
    g = rng(sum(shape))
    a = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-9, 9, shape, generator=g).float())
    check_quantized(a.to(dtype).to(DEV))


def test_quantize_every_bf16_number_in_every_place_of_a_step():
    """Each number alone in a block with one that sets the scale: every rounding, ties and the range beyond 6 included."""
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(BF16)
    a = torch.zeros(1 << 16, 32, dtype=BF16)
    a[:, 5] = bits
    a[:, 9] = torch.where(torch.isfinite(bits), bits, torch.ones_like(bits)) * 0.3
    check_quantized(a.to(DEV))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_quantize_ties_and_neighbours(dtype):
    middles = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], dtype=dtype)
    near = torch.cat([middles, torch.nextafter(middles, torch.zeros_like(middles)), torch.nextafter(middles, middles * 2)])
    a = torch.zeros(2 * near.numel() * 8, 32, dtype=dtype)
    row = 0
    for sign in (1, -1):
        for power in range(-4, 4):
            for x in near:
                a[row, 3], a[row, 31] = sign * x * 2.0 ** power, 4 * 2.0 ** power
                row += 1
    check_quantized(a.to(DEV))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantize_extremes(dtype):
    info = torch.finfo(dtype)
    a = torch.zeros(12, 64, dtype=dtype)
    a[1, 7] = info.max
    a[2] = info.smallest_normal
    a[3, 40] = info.smallest_normal * info.eps     # the smallest denormal number
    a[4] = -0.0
    a[5, 2], a[5, 35] = float("inf"), 1.0          # one block of two becomes NaN
    a[6, 63] = float("-inf")
    a[7, 0], a[7, 1] = float("nan"), 3.0
    a[8] = torch.linspace(-1, 1, 64) * info.smallest_normal
    a[9] = info.max
    a[10] = torch.linspace(-1, 1, 64).to(dtype) * info.smallest_normal * 7
    a[11, 33] = float("-nan")
    codes, scales = check_quantized(a.to(DEV))
    assert scales[5].tolist()[0] == 255 and scales[5].tolist()[1] != 255
    same_bits(mslk_amd.dequantize_mxfp4(codes, scales, F32), O.values(codes, scales), "read back")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_strides(dtype):
    g = rng(3)
    whole = torch.randn(70, 331, generator=g).to(dtype).to(DEV)
    check_quantized(whole[:, 5:5 + 288])               # rows that begin anywhere
    check_quantized(whole[::3, :320])
    check_quantized(whole.t()[:320:1, :64])            # columns that are not neighbours
    check_quantized(whole[:1, 7:7 + 64].expand(9, 64))
    check_quantized(torch.randn(4, 6, 64, generator=g).to(dtype).to(DEV).transpose(0, 1))


def test_quantize_more_than_one_vector_per_lane():
    a = torch.randn(300, 8192, generator=rng(5)).to(BF16).to(DEV)
    check_quantized(a)
    check_quantized(a[:, :8128])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_many_values_at_once_and_in_parts(dtype):
    """Those of 2^27 bytes and more, which go past the caches, in one piece and with gaps between the rows, against parts of them."""
    gen = torch.Generator(DEV).manual_seed(6)
    whole = torch.randn(16500, 4130, generator=gen, device=DEV).to(dtype)
    for a in (whole[:, :4128].contiguous(), whole[:, 1:4129]):
        codes, scales = mslk_amd.quantize_mxfp4(a)
        parts = [mslk_amd.quantize_mxfp4(p) for p in a.split(1500)]
        assert torch.equal(codes, torch.cat([p[0] for p in parts])) and torch.equal(scales, torch.cat([p[1] for p in parts]))
    assert torch.equal(mslk_amd.dequantize_mxfp4(codes, scales, dtype), torch.cat([mslk_amd.dequantize_mxfp4(*p, dtype) for p in parts]))
    check_quantized(a[8000:8050])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 32), (7, 96), (300, 8192), (2, 3, 64), (0, 32)])
def test_dequantize(shape, dtype):
    codes, scales = operand(shape[:-1], shape[-1], rng(11), low=120, high=134)
    got = mslk_amd.dequantize_mxfp4(*gpu(codes, scales), dtype)
    assert got.dtype == dtype
    same_bits(got, O.values(codes, scales))


def test_dequantize_every_scale_and_code():
    codes = (torch.arange(256)[:, None] * 0 + torch.arange(16)[None]).to(torch.uint8)
    codes = codes | (codes.flip(1) << 4)
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8)[:, None]
    for dtype in (F32, BF16):
        same_bits(mslk_amd.dequantize_mxfp4(*gpu(codes, scales), dtype), O.values(codes, scales), str(dtype))


# ---------------------------------------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 32), (1, 8, 64), (3, 17, 96), (16, 64, 256), (17, 130, 288), (33, 256, 512), (64, 128, 1024), (65, 100, 544), (100, 257, 768),
          (128, 384, 2048), (129, 1000, 160), (200, 129, 4096), (256, 256, 512), (257, 511, 1056), (300, 520, 640), (1, 2048, 4096), (20, 512, 2880),
          (513, 768, 1536)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_exact(m, n, k):
    g = rng(m * 7 + n * 3 + k)
    xq, xs = operand(m, k, g)
    wq, ws = operand(n, k, g)
    want, size = O.product(xq, wq, xs, ws)
    assert size.max() < 1 << 20
    same_bits(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws)), want)
    same_bits(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws), out_dtype=F16), want, "fp16")
    for dtype in (F32, BF16):
        bias = torch.randint(-64, 65, (n,), generator=g).to(dtype)
        same_bits(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws), bias=bias.to(DEV)), want + bias.double(), "bias")


@pytest.mark.parametrize("m,n,k", [(1, 100, 4096), (50, 300, 5152), (300, 300, 4096), (700, 512, 14336)])
def test_product_of_wide_scales(m, n, k):
    g = rng(m + n + k)
    xq, xs = operand(m, k, g, 117, 134)
    wq, ws = operand(n, k, g, 110, 125)
    want, size = O.product(xq, wq, xs, ws)
    within(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws)), want, (k / 64 + 64) * 2.0 ** -23 * size)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gated(m, n, k):
    g = rng(m + n * 5 + k)
    xq, xs = operand(m, k, g)
    wq, ws = operand(2 * n, k, g)
    ws -= 7   # sums of a few units, where the sigmoid is neither 0 nor 1
    want, (gate, up, size_gate, size_up) = O.gated(xq, wq, xs, ws)
    assert size_gate.max() < 1 << 13   # sums are exact; left are exp, 1 + e, its reciprocal and two products: 2^-20 is plenty
    # (exp(-gate) in fp32 is off by |gate| 2^-24 for its argument times log2(e), and two units)
    within(mslk_amd.mxfp4_gated_mm(*gpu(xq, wq, xs, ws)), want, (2.0 ** -20 + gate.abs() * 2.0 ** -22) * want.abs() + 1e-37)
    within(mslk_amd.mxfp4_gated_mm(*gpu(xq, wq, xs, ws), out_dtype=F16), want, (2.0 ** -20 + gate.abs() * 2.0 ** -22) * want.abs() + 1e-37)


def test_gated_far_gates():
    """Gates beyond the range of exp, infinite and NaN ones: x = 1 in one channel, gates and their partners in the weights."""
    k = 32
    xq = torch.zeros(2, 16, dtype=torch.uint8)
    xq[:, 0] = 2                                             # 1.0 in channel 0
    xs = torch.full((2, 1), 127, dtype=torch.uint8)
    xs[1] = 0                                                # row 1: 2^-127
    powers = [0, 1, 64, 120, 127, 131, 133, 134, 150, 200, 253]
    wq = torch.zeros(2 * 2 * len(powers), 16, dtype=torch.uint8)
    ws = torch.full((2 * 2 * len(powers), 1), 127, dtype=torch.uint8)
    for i, p in enumerate(powers):
        for sign in (0, 1):
            wq[2 * i + sign, 0], ws[2 * i + sign] = 2 | (sign << 3), p
            wq[2 * len(powers) + 2 * i + sign, 0] = 3        # 1.5
    got = mslk_amd.mxfp4_gated_mm(*gpu(xq, wq, xs, ws)).cpu().double()
    x, w = O.values(xq, xs), O.values(wq, ws)
    gate, up = (x @ w.t())[:, : 2 * len(powers)], (x @ w.t())[:, 2 * len(powers):]
    want = gate * torch.sigmoid(gate) * up
    assert torch.isfinite(got).all()
    # below 2^-126 products of denormal factors may be flushed
    assert ((got - want).abs() <= want.abs() * (2.0 ** -8 + gate.abs().clamp(max=100) * 2.0 ** -22) + 2.0 ** -125).all()
    ws[3] = 255                                              # a NaN gate
    got = mslk_amd.mxfp4_gated_mm(*gpu(xq, wq, xs, ws)).cpu()
    assert torch.isnan(got[:, 3]).all() and torch.isfinite(got[:, :3]).all()


@pytest.mark.parametrize("m,n,k", [(5, 70, 288), (70, 300, 1024), (300, 300, 544)])
def test_nan_scales_stay_in_their_row_and_column(m, n, k):
    """Also those of blocks in the last, shorter step, and with codes of zero."""
    g = rng(k)
    xq, xs = operand(m, k, g)
    wq, ws = operand(n, k, g)
    xs[m // 2, -1] = 255
    ws[n - 1, 0] = 255
    wq[n - 1] = 0
    want, _ = O.product(xq, wq, xs, ws)
    assert torch.isnan(want).sum() == m + n - 1
    same_bits(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws)), want)


def test_empty_products():
    for m, n, k in [(0, 5, 64), (5, 0, 64), (4, 6, 0)]:
        xq, xs = operand(m, k, rng(1))
        wq, ws = operand(n, k, rng(2))
        y = mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws))
        assert y.shape == (m, n) and (y == 0).all()
    bias = torch.arange(6, dtype=F32, device=DEV)
    y = mslk_amd.mxfp4_mm(*gpu(*(operand(4, 0, rng(1))[0], operand(6, 0, rng(1))[0], operand(4, 0, rng(1))[1], operand(6, 0, rng(1))[1])), bias=bias)
    assert torch.equal(y.float(), bias.expand(4, 6))
    xq, xs = operand(4, 0, rng(1))
    wq, ws = operand(6, 0, rng(1))
    assert (mslk_amd.mxfp4_gated_mm(*gpu(xq, wq, xs, ws)) == 0).all()


def test_leading_dimensions_torch_types_and_views():
    g = rng(8)
    xq, xs = gpu(*operand((3, 5), 256, g))
    wq, ws = gpu(*operand(40, 256, g))
    want = O.product(xq, wq, xs, ws)[0].view(3, 5, 40)
    same_bits(mslk_amd.mxfp4_mm(xq, wq, xs, ws), want)
    same_bits(mslk_amd.mxfp4_mm(xq.view(torch.float4_e2m1fn_x2), wq.view(torch.float4_e2m1fn_x2), xs.view(torch.float8_e8m0fnu),
                                ws.view(torch.float8_e8m0fnu)), want, "torch types")
    # codes that begin inside 16 bytes, scales with a stride and with an odd address
    held = torch.zeros(xq.numel() + 8, dtype=torch.uint8, device=DEV)
    held[8:] = xq.flatten()
    strided = torch.zeros(40, 11, dtype=torch.uint8, device=DEV)
    strided[:, 3:] = ws
    same_bits(mslk_amd.mxfp4_mm(held[8:].view(xq.shape), wq, xs, strided[:, 3:]), want, "views")
    long_x, long_xs = gpu(*operand(15, 1024, g))
    long_w, long_ws = gpu(*operand(40, 1024, g))
    odd = torch.zeros(long_xs.numel() + 1, dtype=torch.uint8, device=DEV)
    odd[1:] = long_xs.flatten()
    same_bits(mslk_amd.mxfp4_mm(long_x, long_w, odd[1:].view(long_xs.shape), long_ws), O.product(long_x, long_w, long_xs, long_ws)[0], "odd address")
    one = mslk_amd.mxfp4_mm(xq[0, 0], wq, xs[0, 0], ws)   # a single row without leading dimensions
    assert one.shape == (40,)
    same_bits(one, want[0, 0])


# Sizes for each kind of tile, beside those of few rows above (on 256 CUs): 32 x 32, 32 x 64 and 64 x 64 tiles whose waves take the steps in turn, with
# fewer steps than waves, as many and some more; 128 x 128 tiles; 256-column tiles in less than a round, in a last one that is cut in two (the
# last rows have no second half), with 64, 128, 192 and 256 rows in the last tile.  K from one step to several, whole ones and not.
TILED = [(5, 9000, 288), (32, 8200, 96), (40, 2000, 1280), (128, 1024, 2336), (70, 64, 4096), (1, 64, 2048),
         (520, 1100, 32), (520, 1104, 512), (513, 1100, 800), (33, 20000, 1056),
         (1100, 2000, 224), (1100, 2000, 512), (1025, 2056, 1312), (1, 40000, 64), (2600, 7000, 256),
         (1500, 6000, 288), (1472, 6144, 512), (2600, 7000, 544), (4100, 4200, 800), (4240, 4096, 1024), (4050, 4360, 1056), (3, 70000, 512), (40, 66000, 320),
         (8, 300, 8224), (16, 2000, 5152), (32, 100, 12320), (9, 40, 4128),
         (100, 2600, 1312), (64, 8192, 544), (97, 2621, 2048), (128, 4096, 512), (100, 2602, 64), (32, 16384, 512), (30, 16380, 1056),
         (17, 130, 128), (33, 300, 384), (128, 1024, 2432), (100, 2600, 1408), (300, 1000, 640), (520, 1104, 1920), (2, 2000, 11008)]   # (then: weights streamed, several rounds of pairs; 32 x 64 tiles again; as many 32 x 32 ones as there can be; scales by four bytes, to every end of a pair)


@pytest.mark.parametrize("m,n,k", TILED)
def test_product_exact_with_every_tile(m, n, k):
    g = rng(m + n + k)
    xq, xs = operand(m, k, g)
    wq, ws = operand(n, k, g)
    want, size = O.product(xq, wq, xs, ws)
    assert size.max() < 1 << 20
    args = gpu(xq, wq, xs, ws)
    same_bits(mslk_amd.mxfp4_mm(*args), want)
    for bias_dtype, out_dtype in ((F32, F16), (BF16, BF16)):
        bias = torch.randint(-64, 65, (n,), generator=g).to(bias_dtype)
        same_bits(mslk_amd.mxfp4_mm(*args, bias=bias.to(DEV), out_dtype=out_dtype), want + bias.double(), "bias")
    if n % 2 == 0:
        halves = args[3].view(2, n // 2, -1)
        halves -= 7
        want, (gate, up, _, _) = O.gated(xq, wq, xs, ws - 7)
        within(mslk_amd.mxfp4_gated_mm(*args), want, (2.0 ** -20 + gate.abs() * 2.0 ** -22) * want.abs() + 1e-37, "gated")


@pytest.mark.parametrize("m,n,k", [(40, 2000, 1024), (520, 1104, 512), (1100, 2000, 544), (2600, 7000, 512)])
def test_unaligned_results_bias_and_scales(m, n, k):
    """Addresses that are no multiple of 16 bytes, of everything but the codes, through the C interface."""
    L = _lib.lib()
    g = rng(m + k)
    xq, xs = operand(m, k, g)
    wq, ws = operand(n, k, g)
    bias = torch.randint(-9, 10, (n,), generator=g).to(BF16)
    want, _ = O.product(xq, wq, xs, ws)

    def moved(t, by):
        flat = torch.zeros(t.numel() + by, dtype=t.dtype, device=DEV)
        flat[by:] = t.flatten().to(DEV)
        return flat[by:]

    xs_at, ws_at, bias_at = moved(xs, 1), moved(ws, 3), moved(bias, 1)
    held = torch.full((m * n + 2,), 77.0, dtype=BF16, device=DEV)
    y = held[1:]
    room = L.mslk_amd_mxfp4_mm_workspace_bytes(m, n, k, 0, 0)
    space = torch.empty(max(room, 16), dtype=torch.uint8, device=DEV)
    args = gpu(xq, wq)
    _lib.check(L.mslk_amd_mxfp4_mm(args[0].data_ptr(), args[1].data_ptr(), xs_at.data_ptr(), ws_at.data_ptr(), bias_at.data_ptr(), 2, 0, y.data_ptr(), 0, m, n,
                                   k, space.data_ptr(), space.numel(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    same_bits(y[:-1].view(m, n), want + bias.double())
    assert held[0] == 77 and held[-1] == 77


@pytest.mark.parametrize("m,n,k", [(100, 2000, 4096), (520, 1104, 5152), (1100, 2000, 2080), (1472, 6144, 1056)])
def test_wide_scales_with_every_tile(m, n, k):
    g = rng(m + n + k)
    xq, xs = operand(m, k, g, 117, 134)
    wq, ws = operand(n, k, g, 110, 125)
    want, size = O.product(xq, wq, xs, ws)
    within(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws)), want, (k / 64 + 64) * 2.0 ** -23 * size)


@pytest.mark.parametrize("m,n,k", [(520, 1100, 288), (1100, 2000, 544), (2600, 7000, 288)])
def test_nan_scales_with_every_tile(m, n, k):
    g = rng(k)
    xq, xs = operand(m, k, g)
    wq, ws = operand(n, k, g)
    xs[m - 1, -1] = 255
    ws[n // 2, 0] = 255
    wq[n // 2] = 0
    want, _ = O.product(xq, wq, xs, ws)
    same_bits(mslk_amd.mxfp4_mm(*gpu(xq, wq, xs, ws)), want)


# ---------------------------------------------------------------------------------------------------------------------
# experts
# ---------------------------------------------------------------------------------------------------------------------
def grouped_oracle(xq, wq, xs, ws, sizes, gated):
    parts, at = [], 0
    for e, n in enumerate(sizes):
        n = max(n, 0)
        args = (xq[at:at + n], wq[e], xs[at:at + n], ws[e])
        parts.append(O.gated(*args)[0] if gated else O.product(*args)[0])
        at += n
    return torch.cat(parts)


SIZES = [[5], [0, 0, 3], [1, 1, 1, 1], [100, 0, 33, 7], [64, 64], [300, 1, 0, 256, 257, 2], [0] * 70 + [3, 0, 130] + [1] * 70, [900, 20]]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("n,k", [(72, 512), (130, 288)])
def test_experts(sizes, n, k, gated):
    g = rng(len(sizes) + n)
    xq, xs = operand(sum(sizes), k, g)
    wq, ws = operand((len(sizes), 2 * n if gated else n), k, g)
    if gated:
        ws -= 7
    want = grouped_oracle(xq, wq, xs, ws, sizes, gated)
    got = mslk_amd.mxfp4_grouped_mm(*gpu(xq, wq, xs, ws), torch.tensor(sizes, device=DEV), gated=gated)
    if not gated:
        return same_bits(got, want)
    within(got, want, 2.0 ** -17 * want.abs() + 1e-37)   # gates of at most a few hundred: see test_gated
    each = torch.cat([mslk_amd.mxfp4_gated_mm(*gpu(x, wq[e], s, ws[e])) for e, (x, s) in enumerate(zip(xq.split(sizes), xs.split(sizes))) if len(x)])
    assert torch.equal(got, each)


# Tiles of 64 x 128 (few rows, a K of one step) and the walk over a list of row tiles: more groups than a wave and a workgroup have lanes,
# row tiles of every number of fragments, groups of no rows at both ends, several rounds.
TILED_SIZES = [([1, 0, 3, 0] * 10, 900, 288), ([300, 1, 0, 256, 257, 2], 2000, 160), ([300, 1, 0, 256, 257, 2], 2000, 288), ([0] * 70 + [3, 0, 130] + [1] * 70, 400, 512),
               ([1, 0, 2, 0, 0, 1] * 50, 200, 544), ([0, 64, 65, 128, 129, 192, 193, 255, 256, 257, 0], 2000, 512), ([2000, 0, 1500, 513], 4096, 768),
               ([20, 0, 9, 1], 8320, 4096), ([0] * 70 + [3, 0, 130] + [1] * 70, 1200, 512), ([1, 0, 2, 0, 0, 1] * 50, 800, 544)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes,n,k", TILED_SIZES, ids=lambda v: f"{len(v)}x{sum(v)}" if isinstance(v, list) else str(v))
def test_experts_with_every_tile(sizes, n, k, gated):
    n = n // 2 if gated else n
    g = rng(len(sizes) + n)
    xq, xs = operand(sum(sizes), k, g)
    wq, ws = operand((len(sizes), 2 * n if gated else n), k, g)
    if gated:
        ws -= 7
    want = grouped_oracle(xq, wq, xs, ws, sizes, gated)
    args = gpu(xq, wq, xs, ws)
    counts = torch.tensor(sizes, device=DEV)
    got = mslk_amd.mxfp4_grouped_mm(*args, counts, gated=gated)
    if gated:
        within(got, want, 2.0 ** -17 * want.abs() + 1e-37)
    else:
        same_bits(got, want)
    assert torch.equal(mslk_amd.mxfp4_grouped_mm(*args, counts, gated=gated), got)


def test_no_experts():
    xq, xs = gpu(*operand(5, 64, rng(2)))
    wq, ws = gpu(*operand((0, 6), 64, rng(2)))
    assert mslk_amd.mxfp4_grouped_mm(xq, wq, xs, ws, torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (5, 6)


def call_grouped(xq, wq, xs, ws, sizes, y, gated=False):
    L = _lib.lib()
    G, n, total, k = wq.shape[0], wq.shape[1] // (2 if gated else 1), xq.shape[0], 2 * xq.shape[1]
    room = L.mslk_amd_mxfp4_grouped_mm_workspace_bytes(G, total, n, k, gated, 0)
    space = torch.empty(max(room, 16), dtype=torch.uint8, device=DEV)
    _lib.check(L.mslk_amd_mxfp4_grouped_mm(xq.data_ptr(), wq.data_ptr(), xs.data_ptr(), ws.data_ptr(), sizes.data_ptr(), G, gated, y.data_ptr(),
                                           0 if y.dtype == BF16 else 1, total, n, k, space.data_ptr(), space.numel(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()


@pytest.mark.parametrize("sizes", [[3, 0, 100], [0, 0, 0], [-5, 40, -1], [50, 1 << 40, 7], [300, 300, 300]])
def test_rows_of_no_expert_stay_and_sizes_beyond_the_rows_end_with_them(sizes):
    n, k, total = 72, 512, 200
    g = rng(17)
    xq, xs = operand(total, k, g)
    wq, ws = operand((3, n), k, g)
    y = torch.full((total + 4, n), 77.0, dtype=BF16, device=DEV)
    call_grouped(*gpu(xq, wq, xs, ws), torch.tensor(sizes, device=DEV), y[:total])
    left, clipped = total, []
    for s in sizes:
        clipped.append(min(max(s, 0), left))
        left -= clipped[-1]
    same_bits(y[: total - left], grouped_oracle(xq, wq, xs, ws, clipped, False))
    assert (y[total - left:] == 77).all()


@pytest.mark.parametrize("sizes", [[3, 0, 100, 0], [0, 0, 0, 0], [-5, 90, -1, 70], [50, 1 << 40, 7, 1], [1 << 62, 1 << 62, 1 << 62, 1 << 62], [300, 300, 300, 300]])
@pytest.mark.parametrize("n,k", [(6000, 512), (6000, 160)], ids=["listed", "looked_up"])
def test_sizes_that_do_not_fit_with_every_tile(sizes, n, k):
    total = 280
    g = rng(19)
    xq, xs = operand(total, k, g)
    wq, ws = operand((4, n), k, g)
    y = torch.full((total + 4, n), 77.0, dtype=BF16, device=DEV)
    call_grouped(*gpu(xq, wq, xs, ws), torch.tensor(sizes, device=DEV), y[:total])
    left, clipped = total, []
    for s in sizes:
        clipped.append(min(max(s, 0), left))
        left -= clipped[-1]
    same_bits(y[: total - left], grouped_oracle(xq, wq, xs, ws, clipped, False))
    assert (y[total - left:] == 77).all()


# Operands and results of more than 2^32 bytes, with the kernels that each size takes; looked at are rows and columns from all over.
@pytest.mark.parametrize("m,n,k,gated", [(3, 300000, 32768, False), (300000, 3, 32768, False), (70000, 70000, 288, False), (66000, 66000, 64, False),
                                         (40, 140000, 32768, True)])
def test_offsets_beyond_32_bits(m, n, k, gated):
    gen = torch.Generator(DEV).manual_seed(m + n)
    byte = lambda low, high, *shape: torch.randint(low, high, shape, generator=gen, device=DEV, dtype=torch.uint8)  # noqa: E731
    wide = 2 * n if gated else n
    xq, xs, wq, ws = byte(0, 256, m, k // 2), byte(126, 129, m, k // 32), byte(0, 256, wide, k // 2), byte(126 - 7 * gated, 129 - 7 * gated, wide, k // 32)
    assert max(xq.numel(), wq.numel(), 2 * m * n) > 1 << 32
    y = mslk_amd.mxfp4_gated_mm(xq, wq, xs, ws) if gated else mslk_amd.mxfp4_mm(xq, wq, xs, ws)
    some = lambda size: torch.unique(torch.cat([torch.arange(3), torch.randint(0, size, (20,), generator=rng(1)), torch.arange(size - 3, size)]).clamp(0, size - 1))  # noqa: E731
    rows, columns = some(m).to(DEV), some(n).to(DEV)
    got = y[rows][:, columns]
    if gated:
        both = torch.cat([columns, columns + n])
        want, (gate, up, size_gate, size_up) = O.gated(xq[rows], wq[both], xs[rows], ws[both])
        # sums of 32768 products are not exact here (test_product_of_wide_scales); d silu(g) / dg is below 1.1
        off = (k / 64 + 64) * 2.0 ** -23
        within(got, want, (2.0 ** -20 + gate.abs() * 2.0 ** -22) * want.abs() + 1.1 * off * size_gate * (up.abs() + off * size_up) + gate.abs() * off * size_up)
    else:
        want, size = O.product(xq[rows], wq[columns], xs[rows], ws[columns])
        within(got, want, (k / 64 + 64) * 2.0 ** -23 * size)


def test_offsets_beyond_32_bits_of_experts():
    gen = torch.Generator(DEV).manual_seed(5)
    byte = lambda low, high, *shape: torch.randint(low, high, shape, generator=gen, device=DEV, dtype=torch.uint8)  # noqa: E731
    n, k, sizes = 40000, 8192, [100, 0, 0, 30, 1, 0, 0, 0, 0, 200, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 60]
    xq, xs, wq, ws = byte(0, 256, sum(sizes), k // 2), byte(126, 129, sum(sizes), k // 32), byte(0, 256, 30, n, k // 2), byte(126, 129, 30, n, k // 32)
    assert wq.numel() > 1 << 32
    y = mslk_amd.mxfp4_grouped_mm(xq, wq, xs, ws, torch.tensor(sizes, device=DEV))
    columns = torch.arange(0, n, 1999, device=DEV)
    want = grouped_oracle(xq.cpu(), wq[:, columns].cpu(), xs.cpu(), ws[:, columns].cpu(), sizes, False)
    same_bits(y[:, columns], want)


# ---------------------------------------------------------------------------------------------------------------------
# as programs use them
# ---------------------------------------------------------------------------------------------------------------------
def test_captured_products_follow_their_inputs():
    """A feed-forward block and experts in one graph, replayed with other inputs and sizes and eager calls between the replays."""
    g = rng(23)
    k, experts = 288, 6
    w1q, w1s = gpu(*operand(192, k, g))
    wq, ws = gpu(*operand((experts, 64), 96, g))
    w1s -= 8
    x = torch.randn(40, k, generator=g).to(BF16).to(DEV)
    sizes = torch.tensor([7, 0, 20, 3, 10, 0], device=DEV)

    def block():
        h = mslk_amd.mxfp4_gated_mm(*interleave(mslk_amd.quantize_mxfp4(x), (w1q, w1s)))
        return mslk_amd.mxfp4_grouped_mm(*interleave(mslk_amd.quantize_mxfp4(h), (wq, ws)), sizes), h

    def interleave(a, b):
        return a[0], b[0], a[1], b[1]

    block()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block()
    for i, s in enumerate([[7, 0, 20, 3, 10, 0], [40, 0, 0, 0, 0, 0], [0, 1, 2, 3, 4, 30], [6, 6, 6, 6, 6, 10]]):
        x.copy_(torch.randn(40, k, generator=g).to(BF16))
        sizes.copy_(torch.tensor(s))
        for y in held:
            y.fill_(-1)
        graph.replay()
        got = [y.clone() for y in held]
        want = block()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_captured_experts_with_listed_tiles_follow_their_sizes():
    """Two graphs of one program, each with workspaces of its own, replayed in turn: row tiles are listed again in each replay."""
    g = rng(29)
    k, n, experts, total = 544, 2400, 6, 600
    wq, ws = gpu(*operand((experts, n), k, g))
    operands = [gpu(*operand(total, k, g)) for _ in range(2)]
    sizes = [torch.tensor([100] * 6, device=DEV), torch.tensor([600, 0, 0, 0, 0, 0], device=DEV)]
    run = lambda i: mslk_amd.mxfp4_grouped_mm(operands[i][0], wq, operands[i][1], ws, sizes[i])  # noqa: E731
    run(0)
    torch.cuda.synchronize()
    graphs, held = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            held.append(run(i))
    for step, now in enumerate([[100] * 6, [0, 0, 0, 0, 0, 600], [1, 2, 3, 4, 5, 585], [257, 0, 256, 0, 87, 0], [0, 300, 0, 0, 300, 0]]):
        for i in range(2):
            sizes[i].copy_(torch.tensor(now if i == 0 else now[::-1]))
            operands[i][0].copy_(torch.randint(0, 256, (total, k // 2), generator=g, dtype=torch.uint8))
            held[i].fill_(-1)
        for graph in graphs:
            graph.replay()
        got = [y.clone() for y in held]
        for i in range(2):
            assert torch.equal(got[i], run(i)), (step, i)
            counts = sizes[i].tolist()
            same_bits(got[i], grouped_oracle(operands[i][0].cpu(), wq.cpu(), operands[i][1].cpu(), ws.cpu(), counts, False))


def test_on_another_stream_with_memory_of_its_own():
    g = rng(31)
    xq, xs = gpu(*operand(300, 288, g))
    wq, ws = gpu(*operand(500, 288, g))
    want = mslk_amd.mxfp4_mm(xq, wq, xs, ws)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(9):   # K = 288: each call has a workspace; calls of several streams run at once
        with torch.cuda.stream(streams[i % 3]):
            got.append(mslk_amd.mxfp4_mm(xq, wq, xs, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_outside_of_autograd():
    a = torch.randn(4, 64, device=DEV, requires_grad=True)
    codes, scales = mslk_amd.quantize_mxfp4(a)
    y = mslk_amd.dequantize_mxfp4(codes, scales)
    bias = torch.zeros(4, device=DEV, requires_grad=True)
    assert not mslk_amd.mxfp4_mm(codes, codes, scales, scales, bias=bias).requires_grad and not y.requires_grad


def test_refusals():
    g = rng(1)
    xq, xs = gpu(*operand(4, 64, g))
    wq, ws = gpu(*operand(6, 64, g))
    sizes = torch.tensor([4], device=DEV)
    a = torch.zeros(2, 64, device=DEV)
    cases = [
        (lambda: mslk_amd.quantize_mxfp4(a[:, :40]), "multiple of 32"),
        (lambda: mslk_amd.quantize_mxfp4(a.double()), "dtype"),
        (lambda: mslk_amd.quantize_mxfp4(torch.tensor(1.0, device=DEV)), "multiple of 32"),
        (lambda: mslk_amd.dequantize_mxfp4(xq, ws), "one scale per 16 bytes"),
        (lambda: mslk_amd.dequantize_mxfp4(xq, xs, torch.float64), "out_dtype"),
        (lambda: mslk_amd.dequantize_mxfp4(xq.float(), xs), "codes as uint8"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq, xs.float(), ws), "scales of XQ"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq, xs, ws[:5]), "one scale per 16 bytes"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq[:, :16].contiguous(), xs, ws[:, :1].contiguous()), "share K"),
        (lambda: mslk_amd.mxfp4_mm(xq[:, :16], wq, xs, ws), "contiguous"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq[None], xs, ws[None]), "2-D"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq, xs, ws, bias=torch.zeros(5, device=DEV)), "bias"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq, xs, ws, bias=torch.zeros(6, device=DEV, dtype=F16)), "Bias type"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq, xs, ws, out_dtype=F32), "out_dtype"),
        (lambda: mslk_amd.mxfp4_mm(xq, wq, xs.cpu(), ws), "same device"),
        (lambda: mslk_amd.mxfp4_gated_mm(xq, wq[:5], xs, ws[:5]), "as many gate rows"),
        (lambda: mslk_amd.mxfp4_grouped_mm(xq, wq, xs, ws, sizes), "3-D"),
        (lambda: mslk_amd.mxfp4_grouped_mm(xq, wq[None], xs, ws[None], sizes.int()), "int64"),
        (lambda: mslk_amd.mxfp4_grouped_mm(xq, wq[None], xs, ws[None], sizes.expand(2)), "one entry per group"),
        (lambda: mslk_amd.mxfp4_grouped_mm(xq, wq[None], xs, ws[None], sizes.cpu()), "device"),
        (lambda: mslk_amd.mxfp4_grouped_mm(xq, wq[None, :5], xs, ws[None, :5].contiguous(), sizes, gated=True), "as many gate rows"),
    ]
    for i, (call, text) in enumerate(cases):
        with pytest.raises(RuntimeError, match=text):
            call()
            pytest.fail(f"case {i} was accepted")


def test_shape_functions_agree():
    g = rng(2)
    xq, xs = gpu(*operand((2, 4), 64, g))
    wq, ws = gpu(*operand(6, 64, g))
    checks = ("test_schema", "test_faketensor")
    for op, args in [(torch.ops.mslk.quantize_mxfp4, (torch.randn(3, 64, device=DEV),)), (torch.ops.mslk.dequantize_mxfp4, (xq, xs, F16)),
                     (torch.ops.mslk.mxfp4_mm, (xq, wq, xs, ws, torch.zeros(6, device=DEV), F16)), (torch.ops.mslk.mxfp4_gated_mm, (xq, wq, xs, ws)),
                     (torch.ops.mslk.mxfp4_grouped_mm, (xq[0], wq[None], xs[0], ws[None], torch.tensor([4], device=DEV), True))]:
        torch.library.opcheck(op, args, test_utils=checks)
