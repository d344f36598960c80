"""Paths of the 4-bit floating-point kernels that only very large matrices or forced plans take."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import ashqk
from ashqk import _ext
from oracle import fp4_oracle as F
from test_gpu_fp4 import FORMATS, G, check_product, random_operand, rows

pytestmark = pytest.mark.gpu

VP, I64, CI, CF = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float


def needs_memory(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB of device memory")


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gated", [False, True])
def test_the_longest_rows_in_two_launches(fmt, gated):
    """Rows of 2^24 columns: 128 of them reach 2^30 bytes of codes, and a launch takes no more; the last two rows of 130
    come from a second one. Both equal what their rows give alone, read back too."""
    needs_memory(40)
    k = 1 << 24
    x = torch.empty(130, 2 * k if gated else k, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for row in x:
        row.copy_(torch.randn(row.shape[0], generator=g, device="cuda", dtype=torch.float32))
    call = (lambda t: ashqk.silu_mul_quantize_fp4(t, fmt)) if gated else (lambda t: ashqk.quantize_fp4(t, fmt))
    q, first, last = call(x), call(x[:128]), call(x[128:])
    assert torch.equal(q.codes[:128], first.codes) and torch.equal(q.codes[128:], last.codes)
    blocks = k // F.BLOCK[fmt]
    assert torch.equal(q.scales[:1], first.scales)
    assert torch.equal(q.scales[1:].permute(0, 3, 2, 1, 4).reshape(128, blocks)[:2], last.scales.permute(0, 3, 2, 1, 4).reshape(128, blocks)[:2])
    back = ashqk.dequantize_fp4(q, torch.bfloat16)
    assert torch.equal(back[128:], ashqk.dequantize_fp4(last, torch.bfloat16))
    assert torch.equal(back[120:128], ashqk.dequantize_fp4(first, torch.bfloat16)[120:])
    # and the first columns of the last rows, against the oracle
    if not gated:
        code, byte = F.quantize(x[128:, :4096].double().cpu().numpy(), fmt)
        got = F.unpack(q.codes[128:, :2048].cpu().numpy())
        assert np.array_equal(np.where(got == 8, 0, got), np.where(code == 8, 0, code))
        assert np.array_equal(q.scales_rowmajor()[128:, : byte.shape[1]].cpu().numpy(), byte)


def test_codes_whose_rows_lie_as_far_apart_as_they_may():
    """A pitch of 2^24 bytes: the quantiser's second launch starts at row 128; nothing between the rows is written."""
    needs_memory(8)
    m, k, ld = 131, 500, 1 << 24
    lib = ctypes.CDLL(_ext.C_LIBRARY)
    lib.ashqk_quantize_fp4.argtypes = [VP, I64, CI, CI, VP, I64, VP, CI, CI, CI, CF, VP]
    x = rows(m, k, "fp16", 5)
    for fmt in FORMATS:
        want = ashqk.quantize_fp4(x, fmt)
        wide = torch.full((m, ld), 0x5A, dtype=torch.uint8, device="cuda")
        scales = torch.zeros_like(want.scales)
        assert lib.ashqk_quantize_fp4(x.data_ptr(), x.stride(0), 0, 0, wide.data_ptr(), ld, scales.data_ptr(), m, k, FORMATS.index(fmt), 1.0,
                                      torch.cuda.current_stream().cuda_stream) == 0
        far = ashqk.FP4Tensor(wide[:, :256], scales, (m, k), fmt)
        assert torch.equal(far.codes, want.codes) and torch.equal(far.scales_rowmajor(), want.scales_rowmajor())
        assert bool((wide[:, 256:] == 0x5A).all())
        for dtype in (torch.float16, torch.float32):
            assert torch.equal(ashqk.dequantize_fp4(far, dtype), ashqk.dequantize_fp4(want, dtype))
        v = ashqk.dequantize_fp4(want).double()
        check_product(ashqk.fp4_matmul(far, want, torch.bfloat16), v, v)
        del wide, far


@pytest.mark.parametrize("fmt", FORMATS)
def test_reading_back_beyond_two_to_the_31_pieces(fmt):
    """Rows off 16-byte boundaries are written in pieces of eight values, 2^31 to a launch: 898 rows of 2^24 - 3 columns take
    two, the second from row 896 on."""
    needs_memory(60)
    m, k = 898, (1 << 24) - 3
    codes = torch.randint(0, 256, (m, 1 << 23), dtype=torch.uint8, device="cuda")
    nb = (1 << 24) // F.BLOCK[fmt]
    low, high = (119, 125) if fmt == "mxfp4" else (0, 64)
    scales = torch.randint(low, high, (8, nb // 4, 32, 4, 4), dtype=torch.uint8, device="cuda")
    y = ashqk.dequantize_fp4(ashqk.FP4Tensor(codes, scales, (m, k), fmt), torch.float16)
    part = lambda i, j: ashqk.dequantize_fp4(ashqk.FP4Tensor(codes[i:j], scales[i // 128 : i // 128 + 1].contiguous(), (j - i, k), fmt), torch.float16)  # noqa: E731
    assert torch.equal(y[896:], part(896, 898))
    assert torch.equal(y[768:896], part(768, 896))
    code = F.unpack(codes[896:, :2048].cpu().numpy())
    byte = F.untile_scales(scales[7:, : 4096 // F.BLOCK[fmt] // 4].cpu().numpy(), 2, 4096 // F.BLOCK[fmt])
    assert torch.equal(y[896:, :4096].cpu(), torch.from_numpy(F.values(code, byte, fmt)).half())


@pytest.mark.parametrize("cluster", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("ring", [2, 3, 7])
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_split_of_k_of_the_fused_form(cluster, ring, fmt):
    """x quantised inside the product, plain and gated, up to the 32 rows that are sent in bulk copies to slots of their own:
    clusters that divide K evenly and not, rings shorter than a CTA's slice."""
    lib = ctypes.CDLL(_ext.C_LIBRARY)
    assert lib.ashqk_fp4_set_tuning(cluster, ring, 0) == 0
    try:
        for m, n, k in ((1, 140, 2080), (6, 128, 1504), (16, 200, 1100), (17, 130, 2304), (20, 256, 1056), (25, 300, 500), (32, 128, 2500)):
            w, w64 = random_operand(n, k, fmt, n + k)
            for gated in (False, True):
                x = rows(m, 2 * k if gated else k, "bf16", m + k, spread=False)
                bytes_ = ctypes.c_size_t(1)
                assert lib.ashqk_w4a4_workspace_size(m, n, k, FORMATS.index(fmt), int(gated), ctypes.byref(bytes_)) == 0 and bytes_.value == 0  # fused
                q = (ashqk.silu_mul_quantize_fp4 if gated else ashqk.quantize_fp4)(x, fmt, global_scale=G[fmt])
                x64 = ashqk.dequantize_fp4(ashqk.FP4Tensor(q.codes, q.scales, q.shape, fmt)).double() * float(np.float32(G[fmt]))
                y = ashqk.w4a4_linear(x, w, global_scale=G[fmt], gated=gated)
                check_product(y, x64, w64, 2.0**-23)  # the scales' product in fp32
                assert torch.equal(ashqk.w4a4_linear(x, w, global_scale=G[fmt], gated=gated), y)
    finally:
        assert lib.ashqk_fp4_set_tuning(0, 0, 0) == 0
