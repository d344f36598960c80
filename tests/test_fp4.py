"""Microscaled 4-bit formats without a GPU: the oracle, the layout helpers and every refusal."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import ashqk
from ashqk import _ext
from oracle import fp4_oracle as F

FORMATS = ("mxfp4", "nvfp4")


def test_oracle_rounds_to_the_nearest_element_ties_to_even():
    for x, want in ((0.25, 0), (0.2500001, 1), (0.75, 2), (0.7499, 1), (1.25, 2), (1.75, 4), (2.5, 4), (2.51, 5), (3.5, 6),
                    (5.0, 6), (5.01, 7), (6.0, 7), (7.9, 7)):
        assert int(F._round_to_grid(np.array(x), F.VALUES)) == want, x
    rng = np.random.default_rng(0)
    x = rng.uniform(0, 6, 2000)
    assert np.array_equal(F.VALUES[F._round_to_grid(x, F.VALUES)], F.VALUES[np.abs(F.VALUES[None] - x[:, None]).argmin(1)])


def test_oracle_e4m3_agrees_with_torch():
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(F.E4M3, every)
    x = np.random.default_rng(1).uniform(0, 448, 5000).astype(np.float32)
    x[:127] = F.E4M3
    x[127:253] = (F.E4M3[1:] + F.E4M3[:-1]) / 2  # ties
    got = F._round_to_grid(x.astype(np.float64), F.E4M3)
    assert np.array_equal(got, torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_oracle_known_blocks():
    x = np.zeros((1, 32))
    x[0, :4] = 6.0, -3.0, 0.25, 1.0
    code, byte = F.quantize(x, "mxfp4")
    assert byte[0, 0] == 127 and list(code[0, :4]) == [7, 13, 0, 2]          # scale 2^0
    x[0, 0] = 7.99  # the exponent of 7.99 is 2 as well: held to 6
    assert F.quantize(x, "mxfp4")[0][0, 0] == 7
    x[0, 0] = 8.0
    code, byte = F.quantize(x, "mxfp4")
    assert byte[0, 0] == 128 and code[0, 0] == 6
    x[0, 0] = 6 * 448.0
    code, byte = F.quantize(x, "nvfp4")
    assert byte[0, 0] == 126 and byte[0, 1] == 0 and code[0, 0] == 7
    x[0, 3] = np.nan
    assert F.quantize(x, "nvfp4")[1][0, 0] == 0x7F and F.quantize(x, "mxfp4")[1][0, 0] == 0xFF


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (128, 256), (131, 4096), (300, 160)])
def test_from_rowmajor_lays_scales_out_in_tiles(fmt, rows, k):
    rng = np.random.default_rng(rows + k)
    codes = rng.integers(0, 256, (rows, k // 2), dtype=np.uint8)
    byte = rng.integers(0, 127, (rows, k // F.BLOCK[fmt]), dtype=np.uint8)
    q = ashqk.FP4Tensor.from_rowmajor(torch.from_numpy(codes), torch.from_numpy(byte), fmt)
    assert q.shape == (rows, k)
    assert np.array_equal(q.codes.numpy(), codes)
    assert np.array_equal(q.scales.numpy(), F.tile_scales(byte))
    assert np.array_equal(q.scales_rowmajor().numpy(), byte)


def test_from_rowmajor_pads_an_odd_number_of_nvfp4_blocks():
    q = ashqk.FP4Tensor.from_rowmajor(torch.full((2, 24), 255, dtype=torch.uint8), torch.full((2, 3), 56, dtype=torch.uint8), "nvfp4")
    assert q.codes.shape == (2, 32) and int(q.codes[:, 24:].max()) == 0 and q.scales.shape == (1, 1, 32, 4, 4)
    typed = ashqk.FP4Tensor.from_rowmajor(torch.zeros(2, 24, dtype=torch.uint8), torch.ones(2, 3).to(torch.float8_e4m3fn), "nvfp4")
    assert int(typed.scales[0, 0, 0, 0, 0]) == 0x38


def test_from_rowmajor_refuses():
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    for codes, scales, fmt, g in ((u8(2, 24), u8(2, 1), "mxfp4", 1.0), (u8(2, 16), u8(2, 2), "mxfp4", 1.0), (u8(2, 16), u8(3, 1), "mxfp4", 1.0),
                                  (u8(2, 16), u8(2, 1), "int4", 1.0), (u8(2, 16), u8(2, 1), "mxfp4", 2.0), (u8(2, 16), u8(2, 2), "nvfp4", 0.0),
                                  (u8(2, 16), u8(2, 2), "nvfp4", float("nan")), (torch.zeros(2, 16), u8(2, 1), "mxfp4", 1.0),
                                  (u8(2, 16), torch.zeros(2, 1), "mxfp4", 1.0), (u8(2, 0), u8(2, 0), "mxfp4", 1.0)):
        with pytest.raises(AssertionError):
            ashqk.FP4Tensor.from_rowmajor(codes, scales, fmt, g)


def test_global_scale():
    assert ashqk.fp4_global_scale(torch.tensor([1.0, -2688.0])) == 1.0
    assert ashqk.fp4_global_scale(torch.zeros(4)) == 1.0 and ashqk.fp4_global_scale(torch.zeros(0)) == 1.0
    with pytest.raises(AssertionError):
        ashqk.fp4_global_scale(torch.tensor([float("inf")]))


def test_python_entry_points_refuse():
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(AssertionError):
        ashqk.quantize_fp4(x, "fp4")
    with pytest.raises(AssertionError):
        ashqk.quantize_fp4(x, "mxfp4", global_scale=0.5)
    for g in (0.0, -1.0, 1e19, float("inf"), float("nan")):
        with pytest.raises(AssertionError):
            ashqk.quantize_fp4(x, "nvfp4", global_scale=g)
        with pytest.raises(AssertionError):
            ashqk.w4a4_linear(x, ashqk.FP4Tensor(None, None, (8, 64), "nvfp4"), global_scale=g)
    with pytest.raises(AssertionError):
        ashqk.silu_mul_quantize_fp4(x[:, :63])
    q = lambda k, fmt: ashqk.FP4Tensor(None, None, (2, k), fmt)  # noqa: E731
    with pytest.raises(AssertionError):
        ashqk.fp4_matmul(q(64, "mxfp4"), q(64, "nvfp4"))
    with pytest.raises(AssertionError):
        ashqk.fp4_matmul(q(64, "mxfp4"), q(32, "mxfp4"))
    if not torch.cuda.is_available():  # no CPU path: an error, never a host fallback
        with pytest.raises((RuntimeError, NotImplementedError)):
            ashqk.quantize_fp4(x)


def test_fp4_linear_state_and_refusals():
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    w = lambda fmt="nvfp4", g=0.5: ashqk.FP4Tensor(u8(8, 32), u8(1, 1, 32, 4, 4), (8, 64), fmt, g)  # noqa: E731
    layer = ashqk.FP4Linear(w(), torch.zeros(8), input_global_scale=0.25)
    assert (layer.in_features, layer.out_features) == (64, 8) and "nvfp4" in repr(layer)
    other = ashqk.FP4Linear(w(g=1.0), torch.ones(8))
    other.load_state_dict(layer.state_dict())
    assert other.global_scale == 0.5 and other.input_global_scale == 0.25 and float(other.bias.sum()) == 0
    assert other.weight.shape == (8, 64) and other.weight.global_scale == 0.5
    with pytest.raises(AssertionError):
        ashqk.FP4Linear(w(), torch.zeros(7))
    with pytest.raises(AssertionError):
        ashqk.FP4Linear(w("mxfp4", 1.0), input_global_scale=0.5)
    with pytest.raises(AssertionError):
        ashqk.FP4Linear(w("mxfp4", 1.0), torch.zeros(8)).load_state_dict(layer.state_dict())


VP, I64, CI, CF = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
FAKE = 0x10000  # never dereferenced: validation fails first


def _lib():
    lib = ctypes.CDLL(_ext.C_LIBRARY)
    lib.ashqk_fp4_sizes.argtypes = [CI, CI, CI, ctypes.POINTER(I64), ctypes.POINTER(I64)]
    lib.ashqk_quantize_fp4.argtypes = [VP, I64, CI, CI, VP, I64, VP, CI, CI, CI, CF, VP]
    lib.ashqk_dequantize_fp4.argtypes = [VP, I64, VP, VP, I64, CI, CI, CI, CI, CF, VP]
    lib.ashqk_fp4_matmul.argtypes = [VP, I64, VP, VP, I64, VP, VP, I64, CI, CI, CI, CI, CI, CF, VP]
    lib.ashqk_w4a4_linear.argtypes = [VP, I64, CI, CI, CF, VP, I64, VP, CF, VP, I64, CI, CI, CI, CI, VP, ctypes.c_size_t, VP]
    lib.ashqk_w4a4_workspace_size.argtypes = [CI, CI, CI, CI, CI, ctypes.POINTER(ctypes.c_size_t)]
    return lib


def test_c_abi_sizes():
    lib = _lib()
    ld, n = I64(), I64()
    for m, k, fmt, want in ((1, 32, 0, (16, 512)), (1, 33, 0, (32, 512)), (129, 4096, 0, (2048, 2 * 32 * 512)),
                            (128, 4096, 1, (2048, 64 * 512)), (0, 64, 1, (32, 0)), (1, 48, 1, (32, 512)), (1, 1, 1, (16, 512))):
        assert lib.ashqk_fp4_sizes(m, k, fmt, ctypes.byref(ld), ctypes.byref(n)) == 0
        assert (ld.value, n.value) == want, (m, k, fmt)
    for m, k, fmt in ((-1, 32, 0), (1, 0, 0), (1, 32, 2), (1, 32, -1), (1, (1 << 24) + 1, 0)):
        assert lib.ashqk_fp4_sizes(m, k, fmt, ctypes.byref(ld), ctypes.byref(n)) == 1
    size = ctypes.c_size_t()
    for m, n_, k, fmt in ((0, 8, 32, 0), (1, 0, 32, 0), (1, 8, 0, 0), (1, 8, 32, 7)):
        assert lib.ashqk_w4a4_workspace_size(m, n_, k, fmt, 0, ctypes.byref(size)) == 1


def test_c_abi_switches():
    lib = _lib()
    for which, want in ((0, 0), (1, 0), (2, 0), (3, 1), (-1, 1), (0, 0)):
        assert lib.ashqk_set_fp4_kernel(which) == want
    for cluster, ring, want in ((1, 2, 0), (8, 12, 0), (9, 2, 1), (-1, 0, 1), (0, 1, 1), (0, 13, 1), (0, -1, 1), (0, 0, 0)):
        assert lib.ashqk_fp4_set_tuning(cluster, ring, 0) == want
    for split, want in ((1, 0), (2, 0), (3, 1), (4, 1), (-1, 1), (0, 0)):
        assert lib.ashqk_fp4_set_tuning(0, 0, split) == want


def _refusals(good: dict, bad: list):
    """Each bad change alone must be refused as an invalid argument."""
    for change in bad:
        yield list({**good, **change}.values()), change


def test_c_abi_refuses_before_the_device():
    lib = _lib()
    quant = dict(x=FAKE, x_ld=64, dtype=0, gated=0, codes=FAKE, codes_ld=32, scales=FAKE, M=2, K=64, format=0, g=1.0, stream=None)
    for args, why in _refusals(quant, [{"x": None}, {"x": FAKE + 1}, {"x_ld": 63}, {"dtype": 3}, {"dtype": -1}, {"gated": 1}, {"codes": None},
                                       {"codes": FAKE + 8}, {"codes_ld": 16}, {"codes_ld": 40}, {"scales": None}, {"scales": FAKE + 4},
                                       {"M": 0}, {"M": -1}, {"K": 0}, {"K": 1 << 25, "x_ld": 1 << 25, "codes_ld": 1 << 24}, {"format": 2}, {"g": 2.0}, {"format": 1, "g": 0.0},
                                       {"format": 1, "g": float("nan")}, {"dtype": 2, "x": FAKE + 2}]):
        assert lib.ashqk_quantize_fp4(*args) == 1, why
    dequant = dict(codes=FAKE, codes_ld=32, scales=FAKE, out=FAKE, out_ld=64, dtype=0, M=2, K=64, format=0, g=1.0, stream=None)
    for args, why in _refusals(dequant, [{"codes": None}, {"codes_ld": 24}, {"scales": None}, {"out": None}, {"out_ld": 63}, {"dtype": 9},
                                         {"M": 0}, {"K": 0}, {"format": 5}, {"g": 0.5}, {"out": FAKE + 1}]):
        assert lib.ashqk_dequantize_fp4(*args) == 1, why
    mm = dict(a=FAKE, a_ld=32, a_s=FAKE, b=FAKE, b_ld=32, b_s=FAKE, y=FAKE, y_ld=8, dtype=0, M=2, N=8, K=64, format=0, alpha=1.0, stream=None)
    for args, why in _refusals(mm, [{"a": None}, {"a_ld": 16}, {"a_s": None}, {"b": FAKE + 2}, {"b_ld": 33}, {"b_s": FAKE + 1}, {"y": None},
                                    {"y": FAKE + 1}, {"y_ld": 7}, {"dtype": 2}, {"M": 0}, {"N": 0}, {"K": -1}, {"format": 2}]):
        assert lib.ashqk_fp4_matmul(*args) == 1, why
    lin = dict(x=FAKE, x_ld=64, dtype=0, gated=0, xg=1.0, w=FAKE, w_ld=32, ws=FAKE, wg=1.0, y=FAKE, y_ld=8, M=64, N=8, K=64, format=0,
               work=FAKE, bytes=1 << 20, stream=None)
    for args, why in _refusals(lin, [{"x": None}, {"x_ld": 32}, {"dtype": 2}, {"gated": 1}, {"xg": 0.5}, {"w": None}, {"w_ld": 8}, {"ws": None},
                                     {"wg": 3.0}, {"y": None}, {"y_ld": 4}, {"M": 0}, {"N": -2}, {"K": 0}, {"format": 3}]):
        assert lib.ashqk_w4a4_linear(*args) == 1, why
    assert lib.ashqk_quantize_fp4(*{**quant, "codes_ld": (1 << 24) + 16}.values()) == 2  # rows too far apart
    assert lib.ashqk_fp4_matmul(*{**mm, "b_ld": 1 << 25}.values()) == 2
    assert lib.ashqk_fp4_matmul(*{**mm, "M": (1 << 30) + 1}.values()) == 2
    assert lib.ashqk_w4a4_linear(*{**lin, "N": (1 << 30) + 1, "y_ld": 1 << 31}.values()) == 2
    for change in ({"work": None}, {"bytes": 100}, {"work": FAKE + 8}):
        assert lib.ashqk_w4a4_linear(*{**lin, **change}.values()) == 3, change
