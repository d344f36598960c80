"""silu(gate) * up as it is quantised, over the whole range of gates."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import ashqk
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CENTRES = (-172.0, -150.0, -120.0, -100.0, -93.0, -90.0, -88.5, -87.5, -86.0, -60.0, -20.0, -3.0, 0.0, 3.0, 20.0, 87.5, 89.0, 170.0, 1000.0)


def silu64(x):
    return x * np.exp(np.minimum(x, 0)) / (1 + np.exp(-np.abs(x)))


def gates_and_ups(k, dtype, seed):
    """One row per centre: gates within 2 of it, ups that bring the result near 1 where the type has such values."""
    rng = np.random.default_rng(seed)
    c = np.array(CENTRES)[:, None]
    gate = c + rng.uniform(-2, 2, (len(CENTRES), k))
    most = {"fp16": 6e4, "bf16": 1e38, "fp32": 1e38}[dtype]
    with np.errstate(divide="ignore"):
        up = rng.standard_normal(gate.shape) * np.minimum(most / 5, 1 / np.maximum(np.abs(silu64(c)), 1e-300)).clip(max=most / 5)
    x = torch.from_numpy(np.concatenate([gate, up], 1)).to(DTYPES[dtype])
    assert bool(torch.isfinite(x).all())
    return x.cuda()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("k", [64, 1000])
def test_gates_of_any_size(fmt, dtype, k):
    """Against 64 bits. The activation is off by at most 2^-20 + 2^-23 |gate| relative (exp(-|gate| / 2) enters twice, each
    time with the rounding of its exponent and of that one's constant, together below 0.8 |gate| 2^-24, and two units of the
    exponential, 2^-22; one unit of the reciprocal, 2^-23; five roundings, 5 * 2^-24), so a scale or a code may
    differ only where that moves a value over a border; results below 2^-116 may vanish."""
    g = 1.0 if fmt == "mxfp4" else 0.0371
    x = gates_and_ups(k, dtype, k)
    m = x.shape[0]
    q = ashqk.silu_mul_quantize_fp4(x, fmt, global_scale=g)
    x64 = x.double().cpu().numpy()
    h = silu64(x64[:, :k]) * x64[:, k:]
    d = 2.0**-20 + 2.0**-23 * np.abs(x64[:, :k])
    tiny = np.where(np.abs(h) < 2.0**-116, 0.0, 1.0)
    blocks = (k + 31) // 32 * 32 // F.BLOCK[fmt]
    byte = F.untile_scales(q.scales.cpu().numpy(), m, blocks)
    low, high = F.quantize(h * (1 - d) * tiny, fmt, g)[1], F.quantize(h * (1 + d), fmt, g)[1]
    assert ((byte >= low) & (byte <= high)).all()
    scale = np.repeat(F.scale_values(byte, fmt) * np.float64(np.float32(g)), F.BLOCK[fmt], 1)[:, :k]
    r = np.divide(np.abs(h), scale, out=np.zeros_like(h), where=scale > 0)
    code = F.unpack(q.codes.cpu().numpy())[:, :k]
    low, high = F._round_to_grid(r * (1 - d) * tiny, F.VALUES), F._round_to_grid(r * (1 + d), F.VALUES)
    assert (((code & 7) >= low) & ((code & 7) <= high)).all()
    nonzero = (code & 7) > 0
    assert np.array_equal((code >= 8)[nonzero], (h < 0)[nonzero])
    if dtype != "fp16":  # rows whose exp(-gate) is beyond fp32 are there
        assert (code[np.array(CENTRES) == -90.0] & 7).any()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_the_fused_form_has_the_same_activation(fmt):
    """Four rows quantised inside the product and by the quantiser: one activation."""
    x = gates_and_ups(512, "bf16", 3)[5:9].contiguous()
    six = torch.zeros(512, 512, dtype=torch.float16, device="cuda").fill_diagonal_(6.0)  # exact in both formats
    y = ashqk.w4a4_linear(x, ashqk.quantize_fp4(six, fmt), gated=True)
    v = ashqk.dequantize_fp4(ashqk.silu_mul_quantize_fp4(x, fmt))
    assert bool((v != 0).any(1).all())
    assert torch.equal(y, (v * 6).bfloat16())
