"""Microscaled 4-bit quantisation and products on the GPU against the oracle.

Quantising and reading back are exact: codes, scale bytes and padding equal the oracle's. A product's
terms are exact in fp32 (two 1-bit mantissas and two scales of at most 3 bits), so what remains are the K
additions, each off by at most one unit in the last place of a partial sum (2^-23 of sum |terms|, which
allows for truncation), and the output's rounding, half a step.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import ashqk
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu

FORMATS = ("mxfp4", "nvfp4")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
G = {"mxfp4": 1.0, "nvfp4": 0.0371}


def rows(m, k, dtype, seed, spread=True):
    """N(0, 1) rows whose scale varies over blocks, with exact zeros and block maxima among them."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((m, k))
    if spread:
        x *= np.exp2(rng.integers(-6, 7, (m, -(-k // 16))).repeat(16, 1)[:, :k])
    x[rng.random((m, k)) < 0.02] = 0
    return torch.from_numpy(x).to(DTYPES[dtype]).cuda()


def check_quantised(q, x64, fmt, g, m, k):
    code, byte = F.quantize(x64, fmt, g)
    assert q.shape == (m, k) and q.format == fmt
    assert np.array_equal(F.untile_scales(q.scales.cpu().numpy(), m, byte.shape[1]), byte)
    tiles = q.scales.shape[1] * 4
    if tiles > byte.shape[1]:  # padding blocks of the matrix's rows
        assert not F.untile_scales(q.scales.cpu().numpy(), m, tiles)[:, byte.shape[1]:].any()
    finite = np.repeat(byte != F.NAN_SCALE[fmt], F.BLOCK[fmt], 1)
    got = F.unpack(q.codes.cpu().numpy())
    # -0 and 0 are one value: a zero's sign bit is not compared
    got, code = np.where(got == 8, 0, got), np.where(code == 8, 0, code)
    assert np.array_equal(got[finite], code[finite])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (3, 17), (5, 100), (129, 64), (33, 4096), (260, 1056), (7, 4103)])
def test_quantize_exact(fmt, dtype, m, k):
    x = rows(m, k, dtype, m * 1000 + k)
    q = ashqk.quantize_fp4(x, fmt, global_scale=G[fmt])
    check_quantised(q, x.double().cpu().numpy(), fmt, G[fmt], m, k)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_special_values(fmt):
    x = torch.zeros(12, 64, dtype=torch.float32)
    x[1] = 1e-45                       # smallest subnormal
    x[2] = 3e38
    x[3, 5] = float("inf")
    x[4, 40] = float("nan")
    x[5, 0], x[5, 1] = float("-inf"), float("nan")
    x[6] = -0.0
    x[7] = 1e-30
    x[8] = 448 * 6 * 4.0               # beyond the largest NVFP4 scale
    x[9] = torch.linspace(-6, 6, 64)
    x[10, ::2] = 0.75                  # ties against a scale of 1
    x[10, 1::2] = 6.0
    x[11] = 2.0 ** -126
    for g in ((1.0,) if fmt == "mxfp4" else (1.0, 2.0**-9, 0.0371)):
        q = ashqk.quantize_fp4(x.cuda(), fmt, global_scale=g)
        check_quantised(q, x.double().numpy(), fmt, g, 12, 64)
        back = ashqk.dequantize_fp4(q).cpu()
        b = F.BLOCK[fmt]
        bad = (~torch.isfinite(x)).view(12, -1, b).any(2).repeat_interleave(b, 1)
        assert torch.equal(torch.isnan(back), bad)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k", [64, 100, 999])
def test_quantize_strided_rows_and_leading_dimensions(fmt, k):
    base = rows(24, k + 13, "bf16", k)
    for x in (base[:, :k], base[:, 5 : 5 + k], base[::3, 1 : k + 1], base[:, :k].t().contiguous().t(), base[:, :k].view(4, 6, k) if base[:, :k].is_contiguous() else base[:, :k].unflatten(0, (4, 6)),
              base[:1, :k].expand(24, k)):
        flat = x.reshape(-1, k)
        check_quantised(ashqk.quantize_fp4(x, fmt), flat.double().cpu().numpy(), fmt, 1.0, flat.shape[0], k)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k", [(1, 32), (2, 1), (129, 100), (40, 4096), (3, 777)])
def test_dequantize_exact(fmt, dtype, m, k):
    rng = np.random.default_rng(m + k)
    kp = -(-k // 32) * 32
    code = rng.integers(0, 16, (m, kp), dtype=np.uint8)
    code[:, k:] = 0
    byte = rng.integers(120, 134, (m, kp // 32), dtype=np.uint8) if fmt == "mxfp4" else rng.integers(0, 127, (m, kp // 16), dtype=np.uint8)
    q = ashqk.FP4Tensor(torch.from_numpy(F.pack(code)).cuda(), torch.from_numpy(F.tile_scales(byte, 255)).cuda(), (m, k), fmt, G[fmt])
    got = ashqk.dequantize_fp4(q, DTYPES[dtype])
    # v * s is exact; times the global scale is one fp32 rounding, then the output's.
    want = torch.from_numpy((F.values(code, byte, fmt).astype(np.float32) * np.float32(G[fmt]))[:, :k]).to(DTYPES[dtype])
    assert got.shape == (m, k) and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("start", [0, 1, 3, 4, 8])
def test_dequantize_into_rows_of_any_alignment(fmt, dtype, start):
    """Rows that start anywhere, of any pitch; what lies between and behind them stays as it was."""
    import ctypes

    from ashqk import _ext

    lib = ctypes.CDLL(_ext.C_LIBRARY)
    vp, i64, ci = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    lib.ashqk_dequantize_fp4.argtypes = [vp, i64, vp, vp, i64, ci, ci, ci, ci, ctypes.c_float, vp]
    t = (torch.float16, torch.bfloat16, torch.float32)[dtype]
    for k, ld in ((1, 1), (7, 11), (32, 33), (100, 104), (250, 256), (333, 335), (1024, 1030)):
        q, v64 = random_operand(5, k, fmt, k)
        buf = torch.full((start + 6 * ld,), 9.0, dtype=t, device="cuda")
        out = buf[start : start + 5 * ld].view(5, ld)
        rc = lib.ashqk_dequantize_fp4(q.codes.data_ptr(), q.codes.stride(0), q.scales.data_ptr(), out.data_ptr(), ld, dtype, 5, k,
                                      FORMATS.index(fmt), 1.0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(out[:, :k], v64.to(t)), (k, ld)
        out[:, :k] = 9.0
        assert bool((buf == 9.0).all()), (k, ld)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_quantize_rows_of_any_alignment(fmt, dtype):
    base = rows(9, 700, dtype, 3)
    for start, k in ((1, 32), (2, 97), (3, 640), (4, 15), (5, 333), (6, 16), (7, 48), (8, 500), (9, 31)):
        x = base[:, start : start + k]
        check_quantised(ashqk.quantize_fp4(x, fmt, global_scale=G[fmt]), x.double().cpu().numpy(), fmt, G[fmt], 9, k)
        if dtype != "fp32":
            w, w64 = random_operand(40, k, fmt, k)
            a, b = ashqk.w4a4_linear(x, w, global_scale=G[fmt]), ashqk.w4a4_linear(x.contiguous(), w, global_scale=G[fmt])
            assert torch.equal(a, b), (start, k)


def test_dequantize_mxfp4_extreme_scales():
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    byte = np.arange(256, dtype=np.uint8)[:, None]
    q = ashqk.FP4Tensor(torch.from_numpy(F.pack(code)).cuda(), torch.from_numpy(F.tile_scales(byte)).cuda(), (256, 32))
    with np.errstate(over="ignore"):
        want = F.values(code, byte, "mxfp4").astype(np.float32)
    np.testing.assert_array_equal(ashqk.dequantize_fp4(q).cpu().numpy(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k", [(1, 32), (4, 12288), (37, 500), (130, 64)])
def test_silu_mul_quantize(fmt, dtype, m, k):
    """Against silu(gate) * up in 64 bits. The kernel's fp32 activation is off by at most 2^-19 relative
    (exp by 2 units and its argument's rounding, |gate| <= 8, a sum, a quotient of 2 units, a product), so a
    code may differ only where that moves a value, or its block's largest, over a border."""
    x = rows(m, 2 * k, dtype, m + k, spread=False)
    q = ashqk.silu_mul_quantize_fp4(x, fmt, global_scale=G[fmt])
    x64 = x.double().cpu().numpy()
    h = x64[:, :k] / (1 + np.exp(-x64[:, :k])) * x64[:, k:]
    d = 2.0**-19
    got_byte = F.untile_scales(q.scales.cpu().numpy(), m, (k + 31) // 32 * 32 // F.BLOCK[fmt])
    low, high = (F.quantize(h * f, fmt, G[fmt])[1] for f in (1 - d, 1 + d))
    assert ((got_byte >= low) & (got_byte <= high)).all()
    # the codes against the scale that was chosen
    scale = np.repeat(F.scale_values(got_byte, fmt) * np.float64(np.float32(G[fmt])), F.BLOCK[fmt], 1)[:, :k]
    r = np.divide(np.abs(h), scale, out=np.zeros_like(h), where=scale > 0)
    got = F.unpack(q.codes.cpu().numpy())[:, :k]
    low, high = (F._round_to_grid(r * f, F.VALUES) for f in (1 - d, 1 + d))
    assert (((got & 7) >= low) & ((got & 7) <= high)).all()
    nonzero = (got & 7) > 0
    assert np.array_equal((got >= 8)[nonzero], (h < 0)[nonzero])


def random_operand(m, k, fmt, seed, g=1.0, pad=0):
    """Codes and scales over their whole ranges (scales within 2^+-6, so that fp16 outputs stay finite)."""
    rng = np.random.default_rng(seed)
    kp = -(-k // 32) * 32
    code = rng.integers(0, 16, (m, kp), dtype=np.uint8)
    code[:, k:] = 0
    nb = kp // F.BLOCK[fmt]
    byte = rng.integers(119, 125, (m, nb), dtype=np.uint8) if fmt == "mxfp4" else rng.integers(0, 64, (m, nb), dtype=np.uint8)
    codes = torch.from_numpy(F.pack(code)).cuda()
    if pad:  # rows further apart than they are long
        wide = torch.full((m, codes.shape[1] + pad), 0x77, dtype=torch.uint8, device="cuda")
        wide[:, : codes.shape[1]] = codes
        codes = wide[:, : codes.shape[1]]
    q = ashqk.FP4Tensor(codes, torch.from_numpy(F.tile_scales(byte, F.NAN_SCALE[fmt])).cuda(), (m, k), fmt, g)
    return q, torch.from_numpy(F.values(code, byte, fmt, g)[:, :k]).cuda()


def check_product(y, a64, b64, slack=0.0):
    want, size = a64 @ b64.t(), a64.abs() @ b64.abs().t()
    eps = torch.finfo(y.dtype).eps / 2
    k = a64.shape[1]
    bound = eps * want.abs() + (k + 16) * 2.0**-23 * size * (1 + eps) + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps + slack * size
    worst = ((y.double() - want).abs() / bound).max().item()
    assert y.shape == want.shape and worst <= 1, worst


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 128, 64), (1, 1, 1), (1, 6144, 4096), (7, 256, 4096), (8, 130, 32), (16, 4096, 1024), (17, 300, 352), (32, 128, 12288),
                                   (33, 127, 96), (64, 640, 2080), (100, 4096, 480), (128, 129, 256), (129, 256, 544), (255, 384, 1024),
                                   (256, 256, 512), (257, 100, 4096), (513, 1024, 700), (700, 24, 160), (1024, 2048, 1024)])
def test_matmul(fmt, m, n, k):
    a, a64 = random_operand(m, k, fmt, m + k)
    b, b64 = random_operand(n, k, fmt, n * 7 + k, 0.125 if fmt == "nvfp4" else 1.0)
    dtype = torch.float16 if (m + n) % 2 == 0 else torch.bfloat16
    check_product(ashqk.fp4_matmul(a, b, dtype), a64, b64)


@pytest.fixture(params=[1, 2], ids=["rows", "pair"])
def forced(request):
    """Each product kernel for sizes that the rule gives to the other."""
    import ctypes

    from ashqk import _ext

    lib = ctypes.CDLL(_ext.C_LIBRARY)
    assert lib.ashqk_set_fp4_kernel(request.param) == 0
    yield request.param
    assert lib.ashqk_set_fp4_kernel(0) == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 300, 96), (128, 128, 64), (129, 513, 288), (256, 256, 256), (600, 520, 1312), (1500, 2900, 512)])
def test_matmul_either_kernel(forced, fmt, m, n, k):
    a, a64 = random_operand(m, k, fmt, m)
    b, b64 = random_operand(n, k, fmt, n * 3)
    check_product(ashqk.fp4_matmul(a, b), a64, b64)


@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_many_tiles_per_pair(fmt):
    """More tiles than the persistent kernel's pairs hold at once, an odd number of them each."""
    m, n, k = 256 * 11 + 5, 256 * 23 + 9, 320
    a, a64 = random_operand(m, k, fmt, 1)
    b, b64 = random_operand(n, k, fmt, 2)
    check_product(ashqk.fp4_matmul(a, b), a64, b64)


@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_each_code_and_scale_place(fmt):
    """One nonzero column at a time: every code, block and row of a scale tile lands where it belongs."""
    m, n, k = 160, 144, 512
    b, b64 = random_operand(n, k, fmt, 3)
    code = np.zeros((m, k), np.uint8)
    code[np.arange(m), (np.arange(m) * 37) % k] = 1 + np.arange(m) % 15
    byte = (120 + np.arange(m * (k // F.BLOCK[fmt])) % 5).reshape(m, -1).astype(np.uint8) if fmt == "mxfp4" else \
        (40 + np.arange(m * (k // F.BLOCK[fmt])) % 23).reshape(m, -1).astype(np.uint8)
    a = ashqk.FP4Tensor(torch.from_numpy(F.pack(code)).cuda(), torch.from_numpy(F.tile_scales(byte, 0x7F)).cuda(), (m, k), fmt)
    a64 = torch.from_numpy(F.values(code, byte, fmt)).cuda()
    check_product(ashqk.fp4_matmul(a, b), a64, b64)
    check_product(ashqk.fp4_matmul(b, a), b64, a64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [5, 300])
def test_matmul_row_strided_codes(fmt, m):
    a, a64 = random_operand(m, 320, fmt, 1, pad=48)
    b, b64 = random_operand(200, 320, fmt, 2, pad=16)
    check_product(ashqk.fp4_matmul(a, b), a64, b64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [3, 200])
def test_matmul_nan_stays_in_its_row_and_column(fmt, m):
    x, w = rows(m, 256, "fp32", 5, spread=False), rows(140, 256, "fp32", 6, spread=False)
    x[2, 100], w[130, 3] = float("nan"), float("inf")
    y = ashqk.fp4_matmul(ashqk.quantize_fp4(x, fmt), ashqk.quantize_fp4(w, fmt))
    want = torch.zeros(m, 140, dtype=torch.bool, device="cuda")
    want[2], want[:, 130] = True, True
    assert torch.equal(torch.isnan(y), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [3, 30, 200])
def test_linear_nan_and_infinity_stay_in_their_rows(fmt, gated, m):
    x = rows(m, 512 if gated else 256, "bf16", 5, spread=False)
    x[1, 100], x[2, 255] = float("nan"), float("inf")
    w, _ = random_operand(140, 256, fmt, 1)
    y = ashqk.w4a4_linear(x, w, gated=gated)
    want = torch.zeros(m, 140, dtype=torch.bool, device="cuda")
    want[1], want[2] = True, True
    assert torch.equal(torch.isnan(y), want)


def test_long_rows_and_far_apart_codes():
    """A row of a million columns, and codes whose rows lie megabytes apart."""
    k = (1 << 20) + 96
    x = rows(2, k, "bf16", 1, spread=False)
    for fmt in FORMATS:
        check_quantised(ashqk.quantize_fp4(x, fmt), x.double().cpu().numpy(), fmt, 1.0, 2, k)
        w, w64 = random_operand(3, k, fmt, 2)
        a, a64 = random_operand(2, k, fmt, 3)
        check_product(ashqk.fp4_matmul(a, w, torch.bfloat16), a64, w64)
        q = ashqk.quantize_fp4(x, fmt)
        v64 = ashqk.dequantize_fp4(q).double()
        check_product(ashqk.w4a4_linear(x, w), v64, w64)
        wide = torch.zeros(130, 1 << 22, dtype=torch.uint8, device="cuda")
        b, b64 = random_operand(130, 512, fmt, 4)
        wide[:, :256] = b.codes
        far = ashqk.FP4Tensor(wide[:, :256], b.scales, b.shape, fmt)
        assert torch.equal(ashqk.dequantize_fp4(far), ashqk.dequantize_fp4(b))
        check_product(ashqk.fp4_matmul(far, b, torch.bfloat16), b64, b64)


LINEAR = [(1, 6144, 4096), (1, 100, 64), (2, 4096, 12288), (4, 129, 96), (8, 1024, 1000), (13, 256, 4103), (16, 512, 2048), (17, 128, 4096), (31, 300, 320),
          (64, 256, 512), (130, 384, 1024), (300, 640, 800)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear(fmt, dtype, m, n, k):
    x = rows(m, k, dtype, m + n, spread=False)
    w, w64 = random_operand(n, k, fmt, n + k, 0.25 if fmt == "nvfp4" else 1.0)
    code, byte = F.quantize(x.double().cpu().numpy(), fmt, G[fmt])
    x64 = torch.from_numpy(F.values(code, byte, fmt, G[fmt])[:, :k]).cuda()
    y = ashqk.w4a4_linear(x, w, global_scale=G[fmt])
    assert y.dtype == x.dtype
    check_product(y, x64, w64, 2.0**-23)  # the scales' product in fp32


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear_gated(fmt, dtype, m, n, k):
    """The gated form multiplies what silu_mul_quantize_fp4 gives, bit for bit."""
    x = rows(m, 2 * k, dtype, m + n + 1, spread=False)
    w, w64 = random_operand(n, k, fmt, n + k)
    q = ashqk.silu_mul_quantize_fp4(x, fmt, global_scale=G[fmt])
    x64 = ashqk.dequantize_fp4(ashqk.FP4Tensor(q.codes, q.scales, q.shape, fmt)).double() * float(np.float32(G[fmt]))
    check_product(ashqk.w4a4_linear(x, w, global_scale=G[fmt], gated=True), x64, w64, 2.0**-23)


@pytest.mark.parametrize("m", [1, 40])
def test_linear_leading_dimensions_and_strides(m):
    w, _ = random_operand(192, 256, "mxfp4", 9)
    base = rows(2 * m, 300, "bf16", 4, spread=False)
    x = base[:, 8:264]
    want = ashqk.w4a4_linear(x.contiguous(), w)
    assert torch.equal(ashqk.w4a4_linear(x, w), want)
    assert torch.equal(ashqk.w4a4_linear(x.unflatten(0, (2, m)), w), want.view(2, m, 192))
    assert torch.equal(ashqk.w4a4_linear(base[:, 7:263].contiguous(), w), ashqk.w4a4_linear(base[:, 7:263], w))
    assert torch.equal(ashqk.w4a4_linear(x[0], w), want[0])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 16, 70, 600])
def test_same_result_every_time(fmt, m):
    w, _ = random_operand(4096, 4096, fmt, 11)
    x = rows(m, 4096, "fp16", 12, spread=False)
    first = ashqk.w4a4_linear(x, w, global_scale=G[fmt])
    for _ in range(5):
        assert torch.equal(ashqk.w4a4_linear(x, w, global_scale=G[fmt]), first)


@pytest.mark.parametrize("cluster", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("ring", [2, 3, 7])
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_split_of_k(cluster, ring, fmt):
    """The rows kernel's plans: clusters that divide K evenly and not, rings shorter than a CTA's slice, every
    instruction width, sums in shared memory of their own and in the ring's."""
    import ctypes

    from ashqk import _ext

    lib = ctypes.CDLL(_ext.C_LIBRARY)
    assert lib.ashqk_fp4_set_tuning(cluster, ring, 0) == 0 and lib.ashqk_set_fp4_kernel(1) == 0
    try:
        for m, n, k in ((1, 300, 2080), (4, 128, 4096), (13, 256, 1500), (30, 200, 2304), (61, 130, 1024), (100, 128, 2080), (200, 256, 1056), (300, 140, 800)):
            b, b64 = random_operand(n, k, fmt, n)
            a, a64 = random_operand(m, k, fmt, m)
            check_product(ashqk.fp4_matmul(a, b), a64, b64)
            if m <= 16:
                x = rows(m, k, "bf16", m, spread=False)
                code, byte = F.quantize(x.double().cpu().numpy(), fmt, G[fmt])
                x64 = torch.from_numpy(F.values(code, byte, fmt, G[fmt])[:, :k]).cuda()
                check_product(ashqk.w4a4_linear(x, b, global_scale=G[fmt]), x64, b64, 2.0**-23)
    finally:
        assert lib.ashqk_fp4_set_tuning(0, 0, 0) == 0 and lib.ashqk_set_fp4_kernel(0) == 0


@pytest.mark.parametrize("split", [1, 2])
@pytest.mark.parametrize("fmt", FORMATS)
def test_pairs_that_split_k(split, fmt):
    """Pair tiles whose K is taken by one pair or two: even and uneven shares, ragged edges, an odd pitch of y."""
    import ctypes

    from ashqk import _ext

    lib = ctypes.CDLL(_ext.C_LIBRARY)
    assert lib.ashqk_fp4_set_tuning(0, 0, split) == 0 and lib.ashqk_set_fp4_kernel(2) == 0
    try:
        for m, n, k in ((256, 256, 1024), (130, 500, 4096), (300, 777, 2400), (1, 24, 1100), (512, 1024, 1300), (250, 256, 12288), (700, 300, 5 * 256)):
            a, a64 = random_operand(m, k, fmt, m)
            b, b64 = random_operand(n, k, fmt, n)
            y = ashqk.fp4_matmul(a, b)
            check_product(y, a64, b64)
            assert torch.equal(ashqk.fp4_matmul(a, b), y)
    finally:
        assert lib.ashqk_fp4_set_tuning(0, 0, 0) == 0 and lib.ashqk_set_fp4_kernel(0) == 0


def test_empty():
    w, _ = random_operand(64, 96, "mxfp4", 1)
    assert ashqk.w4a4_linear(torch.zeros(0, 96, dtype=torch.float16, device="cuda"), w).shape == (0, 64)
    q = ashqk.quantize_fp4(torch.zeros(0, 96, dtype=torch.float16, device="cuda"))
    assert q.shape == (0, 96) and ashqk.dequantize_fp4(q).shape == (0, 96)
    assert ashqk.fp4_matmul(q, w).shape == (0, 64) and ashqk.fp4_matmul(w, q).shape == (64, 0)


def test_refusals():
    w, _ = random_operand(64, 96, "mxfp4", 1)
    x = torch.zeros(2, 96, dtype=torch.float16, device="cuda")
    for call in (lambda: ashqk.w4a4_linear(x[:, :64], w), lambda: ashqk.w4a4_linear(x.float(), w), lambda: ashqk.w4a4_linear(x, w, gated=True),
                 lambda: ashqk.w4a4_linear(x.cpu(), w), lambda: ashqk.quantize_fp4(x.int()), lambda: ashqk.quantize_fp4(x[:, :0]),
                 lambda: ashqk.fp4_matmul(w, w, torch.float32), lambda: ashqk.dequantize_fp4(w, torch.float64),
                 lambda: ashqk.dequantize_fp4(ashqk.FP4Tensor(w.codes, w.scales, (64, 200))),
                 lambda: ashqk.dequantize_fp4(ashqk.FP4Tensor(w.codes, w.scales.cpu(), (64, 96))),
                 lambda: ashqk.dequantize_fp4(ashqk.FP4Tensor(w.codes, w.scales[..., :2], (64, 96))),
                 lambda: ashqk.dequantize_fp4(ashqk.FP4Tensor(w.codes.int(), w.scales, (64, 96))),
                 lambda: ashqk.quantize_fp4(x.clone().requires_grad_()), lambda: ashqk.w4a4_linear(x.clone().requires_grad_(), w)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
    with torch.no_grad():
        assert ashqk.w4a4_linear(x.clone().requires_grad_(), w).shape == (2, 64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 9, 48, 300])
def test_mlp_in_a_graph_on_another_stream(fmt, m):
    """gate_up, the gated activation and down as one captured run on a side stream; replays see new inputs, and
    weights quantised right before their first use are the ones that are used."""
    x = rows(m, 512, "bf16", 1, spread=False)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        wg = rows(1536, 512, "bf16", 2, spread=False)
        wd = rows(512, 768, "bf16", 3, spread=False)
        up = ashqk.quantize_fp4(wg, fmt, global_scale=G[fmt])
        h = ashqk.w4a4_linear(x, up, global_scale=G[fmt])
        down = ashqk.quantize_fp4(wd, fmt, global_scale=G[fmt])
        y = ashqk.w4a4_linear(h, down, global_scale=G[fmt], gated=True)
        two_step = ashqk.fp4_matmul(ashqk.silu_mul_quantize_fp4(h, fmt, global_scale=G[fmt]), down, torch.bfloat16)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            hg = ashqk.w4a4_linear(x, up, global_scale=G[fmt])
            yg = ashqk.w4a4_linear(hg, down, global_scale=G[fmt], gated=True)
    torch.cuda.synchronize()
    q = ashqk.quantize_fp4(x, fmt, global_scale=G[fmt])
    v = lambda t: ashqk.dequantize_fp4(ashqk.FP4Tensor(t.codes, t.scales, t.shape, fmt)).double() * float(np.float32(G[fmt]))  # noqa: E731
    check_product(h, v(q), v(up), 2.0**-23)
    hq = ashqk.silu_mul_quantize_fp4(h, fmt, global_scale=G[fmt])
    check_product(y, v(hq), v(down), 2.0**-23)
    check_product(two_step, v(hq), v(down), 2.0**-23)
    for seed in (5, 6):
        x.copy_(rows(m, 512, "bf16", seed, spread=False))
        graph.replay()
        torch.cuda.synchronize()
        want = ashqk.w4a4_linear(ashqk.w4a4_linear(x, up, global_scale=G[fmt]), down, global_scale=G[fmt], gated=True)
        assert torch.equal(yg, want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 20, 40, 300])
def test_weights_and_inputs_written_right_before_their_use(fmt, m):
    """No wait between writing weights, writing x and multiplying: the product sees both as written."""
    stage = [rows(512, 1024, "bf16", s, spread=False) for s in range(4)]
    xs = [rows(m, 1024, "bf16", 10 + s, spread=False) for s in range(4)]
    w, x = torch.empty_like(stage[0]), torch.empty_like(xs[0])
    q = ashqk.quantize_fp4(stage[0], fmt, global_scale=G[fmt])
    codes, scales = torch.empty_like(q.codes), torch.empty_like(q.scales)
    held = ashqk.FP4Tensor(codes, scales, q.shape, fmt, G[fmt])
    got = []
    for i in range(24):
        w.copy_(stage[i % 4])
        x.copy_(xs[i % 3])
        if i % 2:  # codes rewritten in place by a copy, or a new tensor straight from the quantiser
            new = ashqk.quantize_fp4(w, fmt, global_scale=G[fmt])
            codes.copy_(new.codes)
            scales.copy_(new.scales)
            got.append(ashqk.w4a4_linear(x, held, global_scale=G[fmt]))
        else:
            got.append(ashqk.w4a4_linear(x, ashqk.quantize_fp4(w, fmt, global_scale=G[fmt]), global_scale=G[fmt]))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        qw = ashqk.quantize_fp4(stage[i % 4], fmt, global_scale=G[fmt])
        torch.cuda.synchronize()
        assert torch.equal(y, ashqk.w4a4_linear(xs[i % 3], qw, global_scale=G[fmt])), i


def test_calls_on_several_streams_at_once():
    """Products of both kernels, quantisers and an AWQ layer side by side on four streams: each gives what it gives alone."""
    from oracle import awq_oracle as O

    jobs = []
    for i, (m, n, k, fmt) in enumerate(((1, 4096, 4096, "nvfp4"), (16, 2048, 4096, "mxfp4"), (50, 1024, 8192, "nvfp4"), (100, 1536, 2048, "mxfp4"),
                                        (300, 1024, 8192, "mxfp4"), (700, 2048, 1024, "nvfp4"))):
        w, _ = random_operand(n, k, fmt, i)
        x = rows(m, k, "fp16", i, spread=False)
        jobs.append(lambda x=x, w=w: ashqk.w4a4_linear(x, w))
    xa, qw, qz, s = (torch.from_numpy(t).cuda() for t in O.make_problem(4, 4096, 2048, 128, seed=3))
    jobs.append(lambda: ashqk.w4a16_linear(xa, qw, qz, s))
    xb = xa.repeat(64, 1)
    jobs.append(lambda: ashqk.w4a16_linear(xb, qw, qz, s))
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for r in range(12):
        for i, j in enumerate(jobs):
            with torch.cuda.stream(streams[(i + r) % 4]):
                got.append((i, j()))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i]), i


@pytest.mark.parametrize("fmt", FORMATS)
def test_awq_checkpoint_layers_as_fp4(fmt):
    """``replace_linear_layers`` with a 4-bit float format: each layer multiplies the AWQ weights, quantised again."""
    from ashqk.awq_checkpoint import AWQLayer, replace_linear_layers
    from oracle import awq_oracle as O

    layers, dense = {}, {}
    for i, (name, n, k) in enumerate((("up", 384, 256), ("down", 256, 384))):
        _, qw, qz, s = O.make_problem(1, n, k, 128, seed=i)
        bias = torch.randn(n, dtype=torch.float16, device="cuda") if name == "down" else None
        layers[name] = AWQLayer(*(torch.from_numpy(t).cuda() for t in (qw, qz, s)), bias)
        dense[name] = O.dequantize_awq(qw, qz, s, np.float16).T.astype(np.float64)
    model = torch.nn.Sequential()
    model.add_module("up", torch.nn.Linear(256, 384, bias=False))
    model.add_module("down", torch.nn.Linear(384, 256))
    assert replace_linear_layers(model, layers, fmt) == ["up", "down"]
    x = rows(6, 256, "fp16", 1, spread=False)
    for name in ("up", "down"):
        layer, w = getattr(model, name), dense[name]
        g = float(np.float32(np.abs(w).max() / 2688)) if fmt == "nvfp4" else 1.0
        assert isinstance(layer, ashqk.FP4Linear) and layer.global_scale == g
        check_quantised(layer.weight, w, fmt, g, *w.shape)
        code, byte = F.quantize(x.double().cpu().numpy(), fmt)
        x64, (wc, wb) = F.values(code, byte, fmt), F.quantize(w, fmt, g)
        w64 = torch.from_numpy(F.values(wc, wb, fmt, g)).cuda()
        y = layer(x)
        if layer.bias is None:
            check_product(y, torch.from_numpy(x64).cuda(), w64, 2.0**-23)
        else:  # the bias is added to the rounded product
            assert torch.equal(y, ashqk.w4a4_linear(x, layer.weight) + layer.bias)
        x = y
    torch.testing.assert_close(model(rows(6, 256, "fp16", 1, spread=False)), x, rtol=0, atol=0)


def test_rows_behind_the_output_are_left_alone():
    """The C ABI writes y's M x N values and nothing else: rows behind and columns beside keep what they held."""
    import ctypes

    from ashqk import _ext

    lib = ctypes.CDLL(_ext.C_LIBRARY)
    vp, i64, ci = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    lib.ashqk_fp4_matmul.argtypes = [vp, i64, vp, vp, i64, vp, vp, i64, ci, ci, ci, ci, ci, ctypes.c_float, vp]
    for m, n, ld in ((1, 100, 100), (5, 130, 131), (70, 200, 216), (257, 300, 301), (300, 256, 264)):
        a, a64 = random_operand(m, 256, "nvfp4", m)
        b, b64 = random_operand(n, 256, "nvfp4", n)
        buf = torch.full(((m + 3) * ld,), 7.0, dtype=torch.float16, device="cuda")
        rc = lib.ashqk_fp4_matmul(a.codes.data_ptr(), 128, a.scales.data_ptr(), b.codes.data_ptr(), 128, b.scales.data_ptr(), buf.data_ptr(), ld,
                                  0, m, n, 256, 1, 1.0, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0
        y = buf.view(m + 3, ld)
        check_product(y[:m, :n], a64, b64)
        y[:m, :n] = 7.0
        assert bool((buf == 7.0).all()), (m, n)
    bits = ctypes.c_uint(0)
    assert lib.ashqk_get_device_errors(ctypes.byref(bits), 1) == 0 and bits.value == 0
