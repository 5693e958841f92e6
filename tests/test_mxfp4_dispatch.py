"""Which kernel an MXFP4 product gets: a dry run of the dispatch, without a GPU for the 256 compute units of a whole MI355X."""
import pytest

from tests import test_mxfp4_forms_gpu as forms
from tests import test_mxfp4_gpu as sizes
from tests.helpers import mxfp4_kernel

TABLE = [
    ((1, 8192, 8192), {}, "mx_tiles<32,32,waves=1x1x4> workgroups=256"),
    ((64, 4096, 14336), {}, "mx_tiles<32,32,waves=1x1x4> workgroups=256"),
    ((16, 16384, 4096), {}, "mx_tiles<32,32,waves=1x1x4> workgroups=512"),        # two to a CU, up to 32 rows
    ((16, 4096, 4128), {}, "mx_stream<16,waves=8> workgroups=128"),
    ((16, 4096, 4096), dict(aligned=False), "mx_stream<16,waves=8> workgroups=128"),
    ((64, 8192, 8192), {}, "mx_tiles<32,64,waves=1x1x4> workgroups=256"),
    ((16, 14336, 4096), dict(gated=True), "mx_tiles<64,64,waves=1x1x2> workgroups=448"),
    ((128, 8192, 8192), {}, "mx_tiles<64,64,waves=1x1x4> workgroups=256"),
    ((256, 8192, 8192), {}, "mx_tiles<64,64,waves=1x1x2> workgroups=512"),
    ((500, 8192, 8192), {}, "mx_tiles<128,128,waves=2x2x1> workgroups=256"),
    ((500, 10240, 4096), {}, "mx_walk tiles=80 workgroups=160"),
    ((500, 14336, 2048), {}, "mx_tiles<128,128,waves=2x2x1> workgroups=448"),     # two to a CU, a short K
    ((500, 10240, 8192), {}, "mx_walk tiles=80 workgroups=160"),
    ((4096, 4096, 4096), {}, "mx_walk tiles=256 workgroups=256"),
    ((8192, 8192, 4096), {}, "mx_walk tiles=1024 workgroups=256"),                # 64 steps per CU
    ((8192, 8192, 8192), {}, "arrange_scales + mx_walk tiles=1024 workgroups=256"),   # 128
    ((8192, 28672, 4096), {}, "arrange_scales + mx_walk tiles=3584 workgroups=256"),
    ((2047, 10000, 4128), dict(gated=True), "arrange_scales + mx_walk tiles=632 workgroups=256"),
    ((4096, 4096, 256), {}, "arrange_scales + mx_tiles<128,128,waves=2x2x1> workgroups=1024"),     # one step: not for the walk
    ((600, 1 << 25, 512), {}, "mx_tiles<128,128,waves=2x2x1> workgroups=1310720"),   # columns beyond 2^25: neither
    ((256, 5120, 4096), dict(gated=True, groups=16), "mx_tiles<64,128,waves=2x2x1> groups workgroups=1600"),
    ((8192, 8192, 5120), dict(groups=16), "list_row_tiles + mx_walk groups tiles=1536 workgroups=256"),
    ((32768, 768, 2048), dict(gated=True, groups=128), "list_row_tiles + mx_walk groups tiles=1536 workgroups=256"),
    ((512, 4096, 14336), dict(groups=8), "mx_tiles<64,128,waves=2x2x1> groups workgroups=512"),
    ((4, 4, 0), {}, "mx_tiles<32,32,waves=1x1x4> workgroups=8"),
    ((0, 4, 64), {}, "nothing to launch"),
]


@pytest.mark.parametrize("size,options,want", TABLE)
def test_dispatch_is_pinned(size, options, want):
    assert mxfp4_kernel(*size, **options) == want


def test_dry_run_reports_errors():
    assert mxfp4_kernel(4, 4, 40).startswith("error: ") and mxfp4_kernel(4, 4, 64, groups=-1).startswith("error: ")


DENSE = ["mx_stream<8,waves=8>", "mx_stream<16,waves=8>", "mx_stream<32,waves=8>"] + [
    arranged + name for arranged in ("", "arrange_scales + ")
    for name in ("mx_tiles<32,32,waves=1x1x4>", "mx_tiles<32,64,waves=1x1x4>", "mx_tiles<64,64,waves=1x1x4>", "mx_tiles<64,64,waves=1x1x2>",
                 "mx_tiles<128,128,waves=2x2x1>", "mx_walk")]
GROUPS = [arranged + name + " groups" for arranged in ("", "arrange_scales + ") for name in ("mx_tiles<64,64,waves=1x1x4>", "mx_tiles<64,64,waves=1x1x2>", "mx_tiles<64,128,waves=2x2x1>")]
GROUPS += ["list_row_tiles + mx_walk groups", "arrange_scales with list_row_tiles + mx_walk groups"]


def test_every_kernel_has_a_size_that_is_tested_in_all_forms():
    """fp16 and bf16 results, with and without bias, gated: tests/test_mxfp4_forms_gpu.py runs all of them at each of these sizes."""
    assert {forms.kernel(m, n, k) for m, n, k, _ in forms.FORMS} == set(DENSE)
    assert {forms.kernel(m, n // 2, k, gated=True) for m, n, k, _ in forms.FORMS} == set(DENSE)
    assert {forms.kernel(sum(s), n, k, groups=len(s)) for s, n, k, _ in forms.GROUP_FORMS} == set(GROUPS)
    assert {forms.kernel(sum(s), n // 2, k, gated=True, groups=len(s)) for s, n, k, _ in forms.GROUP_FORMS} == set(GROUPS)
    for m, n, k, name in forms.FORMS:
        assert forms.kernel(m, n, k) == forms.kernel(m, n // 2, k, gated=True) == name
    for s, n, k, name in forms.GROUP_FORMS:
        assert forms.kernel(sum(s), n, k, groups=len(s)) == forms.kernel(sum(s), n // 2, k, gated=True, groups=len(s)) == name


def test_sizes_for_each_kind_of_tile_still_are():
    """Those of tests/test_mxfp4_gpu.py, which were chosen for the kernels that they get."""
    # (tiles of two waves run there with arranged scales only)
    assert {forms.kernel(m, n, k) for m, n, k in sizes.SHAPES + sizes.TILED} == set(DENSE) - {"mx_tiles<64,64,waves=1x1x2>"}
    assert {forms.kernel(sum(s), n, k, groups=len(s)) for s, n, k in sizes.TILED_SIZES} >= {
        "list_row_tiles + mx_walk groups", "arrange_scales with list_row_tiles + mx_walk groups", "arrange_scales + mx_tiles<64,128,waves=2x2x1> groups"}
