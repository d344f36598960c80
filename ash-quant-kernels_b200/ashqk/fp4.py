"""Microscaled 4-bit floating point: MXFP4 and NVFP4 tensors, their quantiser and their products.

Beside the AWQ integers (``quantize_awq``, ``w4a16_linear``), whose weights are 4-bit and whose products
are 16-bit, these hold both operands in a form that the B200 tensor core multiplies as it is.

An element is E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and negatives); a block of a row's columns shares a scale:

    "mxfp4"  32 columns  scale 2^(floor(log2 amax) - 2), held as E8M0
    "nvfp4"  16 columns  scale E4M3(min(448, amax / (6 g))) times the tensor's global scale g

An element is its value over the scale, rounded to nearest even and held to +-6. All of it runs on CUDA
tensors only, on the current stream, allocates through PyTorch and can be captured in a CUDA graph.
No reference counterpart: the reference multiplies 4-bit weights in 16 bits.
"""

from __future__ import annotations

import math
import warnings

import torch

from . import _ext

FP4_FORMATS = ("mxfp4", "nvfp4")
_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_CODE = {"mxfp4": 0, "nvfp4": 1}
_E4M3_MAX, _E2M1_MAX = 448.0, 6.0

_op_cache: dict = {}


def _op(name: str):
    op = _op_cache.get(name)
    if op is None:
        op = _op_cache[name] = getattr(_ext.ops(), name).default
    return op


def _format(fmt: str) -> int:
    code = _CODE.get(fmt)
    assert code is not None, f"format must be one of {FP4_FORMATS}, got {fmt!r}"
    return code


def _check(fmt: str, g: float) -> int:
    """The format's code, after checking it and a global scale for it."""
    code = _format(fmt)
    assert (1e-18 <= g <= 1e18) if code else g == 1.0, \
        f"global_scale {g} out of range (1 for mxfp4, 1e-18 .. 1e18 for nvfp4)"
    return code


class FP4Tensor:
    """A matrix [rows, K] in microscaled 4-bit form: what ``quantize_fp4`` returns and the products take.

    codes   uint8 [rows, ceil(K / 32) * 16]: two elements to a byte, the even column in the low four
            bits; columns from K on are zero; rows may be strided by a multiple of 16 bytes
    scales  uint8 [ceil(rows / 128), ceil(blocks / 4), 32, 4, 4], contiguous, ``blocks`` = K rounded up to 32
            over the block size: the scale of (row, block) lies at
            [row // 128, block // 4, row % 32, row // 32 % 4, block % 4]. Rows and blocks beyond the matrix
            are padding: blocks 0, rows anything.
    """

    __slots__ = ("codes", "scales", "shape", "format", "global_scale")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, format: str = "mxfp4", global_scale: float = 1.0):
        self.codes, self.scales, self.shape = codes, scales, tuple(shape)
        self.format, self.global_scale = format, global_scale

    @staticmethod
    def from_rowmajor(codes: torch.Tensor, scales: torch.Tensor, format: str = "mxfp4", global_scale: float = 1.0) -> "FP4Tensor":
        """From a checkpoint's plain layout: codes uint8 [rows, K / 2], scales [rows, K / block] (uint8, or float8
        of the format's kind; E4M3 scales without a sign). K is a multiple of the block."""
        _check(format, global_scale)
        block = _BLOCK[format]
        assert codes.dtype == torch.uint8 and codes.dim() == 2 and scales.dim() == 2
        rows, k = codes.shape[0], 2 * codes.shape[1]
        if scales.dtype != torch.uint8:
            assert scales.dtype == (torch.float8_e8m0fnu if format == "mxfp4" else torch.float8_e4m3fn)
            scales = scales.view(torch.uint8)
        assert k % block == 0 and k > 0 and scales.shape == (rows, k // block), \
            f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not {format} of one matrix"
        # The tensor core takes E4M3 scales as unsigned, so a sign would count in dequantize_fp4 alone.
        assert format == "mxfp4" or not bool((scales > 127).any()), "nvfp4 scales must not be negative"
        kp = -(-k // 32) * 32
        blocks = kp // block
        codes = torch.nn.functional.pad(codes, (0, (kp - k) // 2)).contiguous()
        tiles, cols = -(-rows // 128), -(-blocks // 4)
        full = scales.new_zeros(tiles * 128, cols * 4)
        full[:rows, : k // block] = scales
        tiled = full.view(tiles, 4, 32, cols, 4).permute(0, 3, 2, 1, 4).contiguous()
        return FP4Tensor(codes, tiled, (rows, k), format, global_scale)

    def scales_rowmajor(self) -> torch.Tensor:
        """The scale bytes as uint8 [rows, ceil(K / block)]."""
        tiles, cols = self.scales.shape[:2]
        flat = self.scales.permute(0, 3, 2, 1, 4).reshape(tiles * 128, cols * 4)
        return flat[: self.shape[0], : -(-self.shape[1] // _BLOCK[self.format])].contiguous()

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __repr__(self) -> str:
        return f"FP4Tensor({self.shape}, {self.format!r}, global_scale={self.global_scale}, device={self.device})"


def fp4_global_scale(x: torch.Tensor) -> float:
    """The NVFP4 global scale that maps the largest magnitude of x onto the largest value of the format
    (amax / (448 * 6)); 1 for a tensor of zeros. Copies one number to the host.

    A global scale is at least 1e-18, which tensors with an amax below 2.7e-15 get (blocks under 6e-21 become 0 with it),
    and at most 1e18: a larger amax than 2.7e21 is an error.
    """
    amax = float(x.detach().abs().amax()) if x.numel() else 0.0
    assert math.isfinite(amax), "x holds an infinity or a NaN"
    if amax == 0.0:
        return 1.0
    g = float(torch.tensor(amax / (_E4M3_MAX * _E2M1_MAX), dtype=torch.float32))
    assert g <= 1e18, f"largest magnitude {amax} is beyond what NVFP4 with a global scale of 1e18 holds"
    return max(g, 1e-18)


def quantize_fp4(x: torch.Tensor, format: str = "mxfp4", *, global_scale: float = 1.0) -> FP4Tensor:
    """x [..., K] (fp16, bf16 or fp32) -> FP4Tensor of shape (rows, K); any K, strided rows as they are.

    ``global_scale`` belongs to "nvfp4" (see ``fp4_global_scale``); a block with an infinity or a NaN
    reads back as NaN.
    """
    codes, scales = _op("quantize_fp4")(x, _check(format, global_scale), global_scale, False)
    return FP4Tensor(codes, scales, (codes.shape[0], x.shape[-1]), format, global_scale)


def silu_mul_quantize_fp4(gate_up: torch.Tensor, format: str = "mxfp4", *, global_scale: float = 1.0) -> FP4Tensor:
    """gate_up [..., 2 K] -> FP4Tensor of silu(gate) * up, gate and up the two halves of the last dimension.

    The activation is computed in fp32, off by at most 2^-20 + 2^-23 |gate| of itself, and then rounded to the format: one
    pass over gate_up.
    """
    k = gate_up.shape[-1]
    assert k % 2 == 0, "gate and up are the two halves of the last dimension"
    codes, scales = _op("quantize_fp4")(gate_up, _check(format, global_scale), global_scale, True)
    return FP4Tensor(codes, scales, (codes.shape[0], k // 2), format, global_scale)


def dequantize_fp4(q: FP4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of q, [rows, K] in fp16, bf16 or fp32."""
    return _op("dequantize_fp4")(q.codes, q.scales, q.shape[1], _format(q.format), q.global_scale, dtype)


def fp4_matmul(a: FP4Tensor, b: FP4Tensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """a [M, K] @ b [N, K]^T in fp32, rounded to fp16 or bf16. Both operands have the same format."""
    assert a.format == b.format, f"operands of two formats: {a.format}, {b.format}"
    assert a.shape[1] == b.shape[1], f"K differs: {a.shape}, {b.shape}"
    return _op("fp4_matmul")(a.codes, a.scales, b.codes, b.scales, a.shape[1], _format(a.format),
                             a.global_scale * b.global_scale, dtype)


def w4a4_linear(x: torch.Tensor, weight: FP4Tensor, *, global_scale: float = 1.0, gated: bool = False) -> torch.Tensor:
    """y = Q(x) @ weight^T: x [..., K] fp16 or bf16 is quantised to the weights' format on the way; y [..., N]
    has x's type.

    ``gated``: x is [..., 2 K] and silu(x[..., :K]) * x[..., K:] takes its place (an MLP's down
    projection). ``global_scale`` is x's, for "nvfp4".
    """
    return _op("w4a4_linear")(x, weight.codes, weight.scales, weight.shape[1], _check(weight.format, global_scale),
                              global_scale, weight.global_scale, gated)


class FP4Linear(torch.nn.Module):
    """A linear layer y = Q(x) @ W^T (+ bias) with W [out, in] held as an ``FP4Tensor``; CUDA only.

    The W4A4 counterpart of ``AWQLinear``; ``gated`` as in ``w4a4_linear``. ``input_global_scale`` is x's, for "nvfp4": take
    ``fp4_global_scale`` of inputs that the layer has seen. With 1 a block of x whose largest magnitude is below 6 * 2^-10
    (0.006) becomes zeros, one below 6 * 2^-6 (0.09) has a scale of less than four bits and one above 2688 is cut off.
    """

    def __init__(self, weight: FP4Tensor, bias: torch.Tensor | None = None, *, input_global_scale: float = 1.0, gated: bool = False):
        super().__init__()
        _check(weight.format, input_global_scale)
        assert bias is None or bias.shape == (weight.shape[0],), f"bias {tuple(bias.shape)} for {weight.shape[0]} outputs"
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach())
        self.out_features, self.in_features = weight.shape
        self.format, self.global_scale = weight.format, weight.global_scale
        self.input_global_scale, self.gated = input_global_scale, gated

    @staticmethod
    def from_float(weight: torch.Tensor, bias: torch.Tensor | None = None, format: str = "nvfp4", **kwargs) -> "FP4Linear":
        """From a dense weight [out, in] on the GPU; for "nvfp4" the global scale is ``fp4_global_scale(weight)``, and
        without an ``input_global_scale`` for x there is a warning."""
        g = fp4_global_scale(weight) if format == "nvfp4" else 1.0
        if format == "nvfp4" and "input_global_scale" not in kwargs:
            warnings.warn("nvfp4 without input_global_scale: with 1, blocks of x below 0.006 become zeros and those above 2688 are "
                          "cut off; pass fp4_global_scale of inputs that the layer has seen", stacklevel=2)
        return FP4Linear(quantize_fp4(weight.detach(), format, global_scale=g), bias, **kwargs)

    @staticmethod
    def from_awq(layer, format: str = "nvfp4", **kwargs) -> "FP4Linear":
        """From an ``AWQLayer`` on the GPU: its int4 weights are dequantised to fp16 and quantised again."""
        w = _op("dequantize_awq")(layer.qweight, layer.qzeros, layer.scales, torch.float16)
        return FP4Linear.from_float(w.t(), layer.bias, format, **kwargs)

    @property
    def weight(self) -> FP4Tensor:
        return FP4Tensor(self.codes, self.scales, (self.out_features, self.in_features), self.format, self.global_scale)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = w4a4_linear(x, self.weight, global_scale=self.input_global_scale, gated=self.gated)
        return y + self.bias.to(y.dtype) if self.bias is not None else y

    def get_extra_state(self):
        return {"format": self.format, "shape": (self.out_features, self.in_features), "global_scale": self.global_scale,
                "input_global_scale": self.input_global_scale}

    def set_extra_state(self, state) -> None:
        assert tuple(state["shape"]) == (self.out_features, self.in_features) and state["format"] == self.format, \
            f"state of {state['shape']} {state['format']} for a layer of {(self.out_features, self.in_features)} {self.format}"
        self.global_scale, self.input_global_scale = state["global_scale"], state["input_global_scale"]

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, format={self.format!r}, "
                f"bias={self.bias is not None}, gated={self.gated}")
