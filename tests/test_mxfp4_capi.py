"""MXFP4 without a GPU: refusals of the C entry points before anything is launched, sizes of workspaces, tensors without data."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mslk_amd
from mslk_amd import _lib

SOMEWHERE = 1 << 20   # a pointer that is not followed
L = _lib.lib()


def error():
    return L.mslk_amd_last_error().decode()


def mm(m=4, n=6, k=64, *, xq=SOMEWHERE, ws=SOMEWHERE, bias=None, bias_dtype=0, gated=0, y=SOMEWHERE, y_dtype=0, workspace=None, size=0):
    return L.mslk_amd_mxfp4_mm(xq, SOMEWHERE, SOMEWHERE, ws, bias, bias_dtype, gated, y, y_dtype, m, n, k, workspace, size, None)


@pytest.mark.parametrize("options,text", [
    (dict(m=-1), "negative"), (dict(k=40), "multiple of 32"), (dict(m=1 << 31), "out of range"), (dict(k=1 << 24), "out of range"),
    (dict(gated=1, n=1 << 20, k=1 << 14), "too large"), (dict(y_dtype=2), "output expected"), (dict(y=None), "null output"),
    (dict(y=SOMEWHERE + 1), "2-byte aligned"), (dict(xq=None), "null pointer"), (dict(xq=SOMEWHERE + 8), "16-byte aligned"), (dict(ws=None), "null pointer"),
    (dict(m=300, n=4096), "workspace"), (dict(m=300, n=4096, workspace=SOMEWHERE, size=64), "workspace"),
    (dict(m=300, n=4096, workspace=SOMEWHERE + 4, size=1 << 30), "workspace"),
    (dict(bias=SOMEWHERE), "disagree"), (dict(bias_dtype=2), "disagree"), (dict(bias=SOMEWHERE, bias_dtype=3), "bias dtype"),
    (dict(bias=SOMEWHERE, bias_dtype=1, gated=1), "no bias")])
def test_products_refuse(options, text):
    assert mm(**options) != 0 and text in error()


@pytest.mark.parametrize("options,text", [(dict(G=-1), "negative"), (dict(sizes=None), "null pointer"), (dict(n=1 << 18, k=2080), "workspace")])
def test_experts_refuse(options, text):
    o = dict(G=3, n=64, k=512, sizes=SOMEWHERE)
    o.update(options)
    rc = L.mslk_amd_mxfp4_grouped_mm(SOMEWHERE, SOMEWHERE, SOMEWHERE, SOMEWHERE, o["sizes"], o["G"], 0, SOMEWHERE, 0, 100, o["n"], o["k"], None, 0, None)
    assert rc != 0 and text in error()


@pytest.mark.parametrize("call,text", [
    (lambda: L.mslk_amd_quantize_mxfp4(SOMEWHERE, 0, 4, 40, 64, SOMEWHERE, SOMEWHERE, None), "multiple of 32"),
    (lambda: L.mslk_amd_quantize_mxfp4(SOMEWHERE, 7, 4, 64, 64, SOMEWHERE, SOMEWHERE, None), "dtype"),
    (lambda: L.mslk_amd_quantize_mxfp4(SOMEWHERE, 0, -4, 64, 64, SOMEWHERE, SOMEWHERE, None), ""),
    (lambda: L.mslk_amd_dequantize_mxfp4(SOMEWHERE, SOMEWHERE, 4, 40, SOMEWHERE, 0, None), "multiple of 32"),
    (lambda: L.mslk_amd_dequantize_mxfp4(SOMEWHERE, SOMEWHERE, 4, 64, SOMEWHERE + 2, 0, None), "misaligned"),
    (lambda: L.mslk_amd_dequantize_mxfp4(None, SOMEWHERE, 4, 64, SOMEWHERE, 0, None), "null pointer")])
def test_quantizers_refuse(call, text):
    assert call() != 0 and text in error()


@pytest.mark.parametrize("m,n,k,gated", [(1, 8192, 8192, 0), (33, 64, 512, 0), (300, 4096, 288, 0), (4096, 4096, 4096, 1), (8192, 28672, 4096, 0),
                                         (1, 1 << 26, 64, 0), (3, 100000, 1056, 1)])
def test_workspaces_hold_both_tensors_of_scales_or_nothing(m, n, k, gated):
    rows = [-(-r // 64) * 64 for r in (m, n * (2 if gated else 1))]
    both = sum(rows) * -(-k // 512) * 16
    for aligned in (0, 1):
        size = L.mslk_amd_mxfp4_mm_workspace_bytes(m, n, k, gated, aligned)
        assert size in (0, both)
        if m > 32 and (k % 512 or not aligned):
            assert size == both


def test_nothing_to_do_wants_nothing():
    assert L.mslk_amd_mxfp4_mm_workspace_bytes(0, 5, 64, 0, 0) == L.mslk_amd_mxfp4_mm_workspace_bytes(5, 0, 64, 0, 0) == 0
    assert mm(m=0, y=None) == 0 and mm(n=0, y=None) == 0
    assert L.mslk_amd_mxfp4_grouped_mm(None, None, None, None, None, 0, 0, SOMEWHERE, 0, 10, 64, 512, None, 0, None) == 0


def test_python_functions_want_gpu_tensors():
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for call in (lambda: mslk_amd.quantize_mxfp4(torch.zeros(4, 64)), lambda: mslk_amd.dequantize_mxfp4(codes, scales),
                 lambda: mslk_amd.mxfp4_mm(codes, codes, scales, scales), lambda: mslk_amd.mxfp4_gated_mm(codes, codes, scales, scales),
                 lambda: mslk_amd.mxfp4_grouped_mm(codes, codes[None], scales, scales[None], torch.tensor([4]))):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()


def test_shapes_of_tensors_without_data():
    with FakeTensorMode():
        x = torch.empty(2, 5, 128, dtype=torch.bfloat16, device="cuda")
        codes, scales = torch.ops.mslk.quantize_mxfp4(x)
        assert codes.shape == (2, 5, 64) and scales.shape == (2, 5, 4) and codes.dtype == scales.dtype == torch.uint8
        assert torch.ops.mslk.dequantize_mxfp4(codes, scales).shape == x.shape
        w, ws = torch.empty(6, 64, dtype=torch.uint8, device="cuda"), torch.empty(6, 4, dtype=torch.uint8, device="cuda")
        assert torch.ops.mslk.mxfp4_mm(codes, w, scales, ws).shape == (2, 5, 6)
        assert torch.ops.mslk.mxfp4_mm(codes, w, scales, ws, None, torch.float16).dtype == torch.float16
        assert torch.ops.mslk.mxfp4_gated_mm(codes, w, scales, ws).shape == (2, 5, 3)
        rows, row_scales, sizes = codes.view(10, 64), scales.view(10, 4), torch.empty(1, dtype=torch.int64, device="cuda")
        assert torch.ops.mslk.mxfp4_grouped_mm(rows, w[None], row_scales, ws[None], sizes, True).shape == (10, 3)
