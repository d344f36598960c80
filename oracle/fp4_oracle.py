"""Microscaled 4-bit floating point in numpy: the definition of the formats, for the tests.

Everything is in 64 bits except the two quotients of NVFP4 (amax / (6 g) and x / scale), which the format's
definition here rounds to fp32 once before they are rounded to E4M3 and E2M1.
"""

from __future__ import annotations

import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"mxfp4": 32, "nvfp4": 16}
NAN_SCALE = {"mxfp4": 0xFF, "nvfp4": 0x7F}


def _round_to_grid(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the nearest value of an ascending grid, ties to the even index, the last beyond it."""
    hi = np.clip(np.searchsorted(grid, x), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    dh, dl = grid[hi] - x, x - grid[lo]
    take_lo = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    return np.where(take_lo, lo, hi)


E4M3 = np.array([(m / 8 * 2.0**-6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def scale_values(byte: np.ndarray, fmt: str) -> np.ndarray:
    if fmt == "mxfp4":
        return np.where(byte == 0xFF, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return np.where(byte == 0x7F, np.nan, E4M3[np.minimum(byte, 126)])


def quantize(x: np.ndarray, fmt: str, g: float = 1.0):
    """x [M, K] -> codes [M, Kp] (0..15, Kp = K up to 32), scale bytes [M, Kp / block]."""
    m, k = x.shape
    b = BLOCK[fmt]
    kp = -(-k // 32) * 32
    blocks = np.zeros((m, kp), np.float64)
    blocks[:, :k] = x
    blocks = blocks.reshape(m, kp // b, b)
    with np.errstate(all="ignore"):
        amax = np.abs(blocks).max(2)
        bad = ~np.isfinite(amax)
        amax = np.where(bad, 1.0, amax)
        if fmt == "mxfp4":
            e = np.where(amax > 0, np.frexp(amax)[1] - 1 - 2, -127)
            byte = np.maximum(e, -127) + 127
            scale = np.exp2(byte - 127.0)
            q = np.abs(blocks) / scale[..., None]
        else:
            g32 = np.float32(g)
            t = amax.astype(np.float32) / (np.float32(6) * g32)
            byte = _round_to_grid(np.minimum(t.astype(np.float64), 448.0), E4M3)
            scale = (E4M3[byte].astype(np.float32) * g32)[..., None]
            q = (np.abs(blocks).astype(np.float32) / np.where(scale > 0, scale, np.float32(1))).astype(np.float64)
            q = np.where(scale > 0, q, 0.0)
        q = np.where(np.isnan(q), 6.0, q)
    code = _round_to_grid(q, VALUES) + 8 * np.signbit(blocks)
    byte = np.where(bad, NAN_SCALE[fmt], byte)
    return code.reshape(m, kp).astype(np.uint8), byte.astype(np.uint8)


def values(code: np.ndarray, byte: np.ndarray, fmt: str, g: float = 1.0) -> np.ndarray:
    """What codes [M, Kp] and scale bytes stand for, in 64 bits."""
    v = VALUES[code & 7] * np.where(code & 8, -1.0, 1.0)
    return v * np.repeat(scale_values(byte, fmt), BLOCK[fmt], 1)[:, : code.shape[1]] * np.float64(np.float32(g))


def pack(code: np.ndarray) -> np.ndarray:
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def unpack(codes: np.ndarray) -> np.ndarray:
    return np.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)


def tile_scales(byte: np.ndarray, fill: int = 0) -> np.ndarray:
    """[M, blocks] -> [ceil(M/128), ceil(blocks/4), 32, 4, 4], one scale at a time; padding rows hold ``fill``."""
    m, nb = byte.shape
    out = np.full((-(-m // 128), -(-nb // 4), 32, 4, 4), fill, np.uint8)
    r, b = np.arange(m)[:, None], np.arange(out.shape[1] * 4)[None]
    full = np.zeros((m, out.shape[1] * 4), np.uint8)
    full[:, :nb] = byte
    out[r // 128, b // 4, r % 32, r // 32 % 4, b % 4] = full
    return out


def untile_scales(tiled: np.ndarray, m: int, nb: int) -> np.ndarray:
    r, b = np.arange(m)[:, None], np.arange(nb)[None]
    return tiled[r // 128, b // 4, r % 32, r // 32 % 4, b % 4]
