"""The microscaled 4-bit floating-point operators, as cases that can be measured.

Operators: ``quantize_fp4`` (with ``dequantize_fp4``, which reads its result back),
``silu_mul_quantize_fp4`` (the gated activation of an MLP, quantised as it is made),
``w4a4_linear`` (16-bit activations quantised on the fly times 4-bit weights, from one token to a
prefill) and ``fp4_matmul`` (the product of two quantised operands).

Formats. An element is E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even
column in the low four bits. A row's columns are cut into blocks that share one scale:

* ``mxfp4``: 32 columns, scale 2^(floor(log2(amax)) - 2) held as E8M0;
* ``nvfp4``: 16 columns, scale amax / (6 g) rounded to E4M3 (at most 448), times a global scale g.

An element is its value over the scale, rounded to nearest even and held to +-6. Rows of codes are
padded with zeros to a multiple of 32 columns. Scales lie in tiles of 128 rows x 4 blocks,
``[row tile, block tile, row % 32, row // 32 % 4, block % 4]``, the order in which the tensor core
takes them. ``run`` computes the operators in plain torch where ``own`` is false and calls the
framework where it is true.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ash-quant-kernels_b200")
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One token's hidden state, quantised and read back: the smallest call, bound by its launch.
        {"name": "quantize decode", "op": "quantize", "m": 1, "k": 4096, "format": "mxfp4", "dtype": "bf16"},
        # A ragged batch of rows whose length ends inside a block.
        {"name": "quantize ragged", "op": "quantize", "m": 509, "k": 4103, "format": "nvfp4", "dtype": "fp16"},
        # A layer's weight matrix, or a long prefill's activations.
        {"name": "quantize large", "op": "quantize", "m": 8192, "k": 12288, "format": "nvfp4", "dtype": "fp16"},
        # The gated activation between gate_up and down, for a few decoded tokens and for a prefill.
        {"name": "gated decode", "op": "gated", "m": 4, "k": 12288, "format": "nvfp4", "dtype": "bf16"},
        {"name": "gated prefill", "op": "gated", "m": 2048, "k": 12288, "format": "mxfp4", "dtype": "fp16"},
        # Decode: the qkv projection of one token, down of four with its gated input, gate_up of sixteen.
        {"name": "linear qkv 1", "op": "linear", "m": 1, "n": 6144, "k": 4096, "format": "nvfp4", "dtype": "fp16"},
        {"name": "linear down 4", "op": "gated_linear", "m": 4, "n": 4096, "k": 12288, "format": "mxfp4", "dtype": "bf16"},
        {"name": "linear gate_up 16", "op": "linear", "m": 16, "n": 24576, "k": 4096, "format": "mxfp4", "dtype": "fp16"},
        # A short prompt or a batch of drafts, an odd number of rows.
        {"name": "linear o 101", "op": "linear", "m": 101, "n": 4096, "k": 4096, "format": "nvfp4", "dtype": "bf16"},
        # Prefill.
        {"name": "linear down 2048", "op": "gated_linear", "m": 2048, "n": 4096, "k": 12288, "format": "nvfp4", "dtype": "bf16"},
        # Operands that are both in hand quantised: an odd number of rows, and the largest product.
        {"name": "matmul qkv 513", "op": "matmul", "m": 513, "n": 6144, "k": 4096, "format": "nvfp4", "dtype": "fp16"},
        {"name": "matmul gate_up 8192", "op": "matmul", "m": 8192, "n": 24576, "k": 4096, "format": "mxfp4", "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("quantize", "gated", "linear", "linear", "gated_linear", "matmul"))
    fmt = rng.choice(("mxfp4", "nvfp4"))
    case = {"op": op, "m": _spread(rng, 1, 8192), "k": _spread(rng, 64, 12288), "format": fmt}
    if rng.random() < 0.6:  # most layers have round sizes, some callers' do not
        case["k"] = max(64, case["k"] // 64 * 64)
    if op == "quantize":
        case["dtype"] = rng.choice(("fp16", "bf16", "fp32"))
        return case
    case["dtype"] = rng.choice(("fp16", "bf16"))
    if op != "gated":
        n = _spread(rng, 64, 24576)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        case["n"] = n
        # At most the largest listed product's work.
        case["m"] = max(1, min(case["m"], 8192 * 24576 * 4096 // (n * case["k"])))
    return case


# ---- inputs ---------------------------------------------------------------------------------------


def _activations(m, k, dtype, g):
    """Values as a normalised hidden state has them: near N(0, 1), a few channels far larger."""
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.float32)
    big = torch.rand(k, generator=g, device="cuda") < 0.004
    return (x * torch.where(big, 20.0, 1.0)).to(dtype)


def _global_scale(case):
    # Calibrated once by a user's program, held in few bits: the largest activations fit E4M3 scales.
    return 1.0 if case["format"] == "mxfp4" else 11 / 256


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, m, k = case["op"], case["m"], case["k"]
    dtype = _TYPES[case["dtype"]]
    state = {"op": op, "format": case["format"], "dtype": dtype, "m": m, "k": k, "g": _global_scale(case)}
    if op in ("quantize", "linear"):
        state["x"] = _activations(m, k, dtype, g)
    elif op in ("gated", "gated_linear"):
        state["x"] = torch.randn(m, 2 * k, generator=g, device="cuda", dtype=torch.float32).to(dtype)
    else:
        state["a"] = _pack(_activations(m, k, dtype, g), case["format"], state["g"])
    if "n" in case:  # the layer's weights, quantised when it was loaded
        n = case["n"]
        state["n"] = n
        state["wg"] = 1.0 if case["format"] == "mxfp4" else 0.1 / (6 * 448)
        state["w"] = _pack(torch.randn(n, k, generator=g, device="cuda", dtype=torch.float32) * 0.02, case["format"], state["wg"])
    return state


def _pack(x, fmt, g):
    """A quantised operand as a program keeps it: (codes, scales)."""
    rows, k = x.shape
    magnitude, negative, byte = _elements(x.float(), fmt, g)[:3]
    kp = -(-k // 32) * 32
    code = torch.zeros(rows, kp, dtype=torch.uint8, device=x.device)
    table = torch.tensor(_VALUES, device=x.device)
    code[:, :k] = (torch.searchsorted(table, magnitude.contiguous()) + 8 * negative)[:, :k].to(torch.uint8)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    blocks = kp // _BLOCK[fmt]
    tiles, cols = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros(tiles * 128, cols * 4, dtype=torch.uint8, device=x.device)
    full[:rows, : byte.shape[1]] = byte
    scales = full.view(tiles, 4, 32, cols, 4).permute(0, 3, 2, 1, 4).contiguous()
    return codes.contiguous(), scales


# ---- the plain form -------------------------------------------------------------------------------


def _elements(x, fmt, g):
    """Rounded magnitudes, signs, the scales' bytes and the scales' values (one per column) of fp32 rows."""
    rows, k = x.shape
    b = _BLOCK[fmt]
    kp = -(-k // b) * b
    if kp != k:
        x = torch.cat([x, x.new_zeros(rows, kp - k)], 1)
    block = x.view(rows, kp // b, b)
    amax = block.abs().amax(2)
    if fmt == "mxfp4":
        exponent = (torch.frexp(amax)[1] - 3).clamp(min=-127)
        exponent = torch.where(amax > 0, exponent, -127)
        byte = (exponent + 127).to(torch.uint8)
        scale = torch.ldexp(torch.ones_like(amax), exponent)
    else:
        held = (amax / (6.0 * torch.tensor(g, device=x.device))).clamp(max=448.0).to(torch.float8_e4m3fn)
        byte = held.view(torch.uint8)
        scale = held.float() * g
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = torch.where((scale > 0)[..., None], block.abs() / safe[..., None], torch.zeros_like(block))
    step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0))
    q = (torch.round(q / step) * step).clamp(max=6.0)
    shape = (rows, kp)
    return q.view(shape), torch.signbit(block).view(shape), byte, scale.repeat_interleave(b, 1)


def _rounded(x, fmt, g):
    """fp32 rows as the format holds them, in fp32."""
    q, negative, _, scale = _elements(x, fmt, g)
    return (torch.where(negative, -q, q) * scale)[:, : x.shape[1]]


def _unpack(packed, fmt, g, k):
    """The values, in fp32, that (codes, scales) stand for."""
    codes, scales = packed
    rows = codes.shape[0]
    code = torch.stack([codes & 15, codes >> 4], 2).view(rows, -1)[:, :k].long()
    value = torch.tensor(_VALUES, device=codes.device)[code & 7]
    value = torch.where(code >= 8, -value, value)
    tiles, cols = scales.shape[:2]
    byte = scales.permute(0, 3, 2, 1, 4).reshape(tiles * 128, cols * 4)[:rows]
    scale = torch.ldexp(torch.ones((), device=codes.device), byte.int() - 127) if fmt == "mxfp4" else byte.contiguous().view(torch.float8_e4m3fn).float() * g
    return value * scale.repeat_interleave(_BLOCK[fmt], 1)[:, :k]


def _silu_mul(x):
    gate, up = x.float().chunk(2, 1)
    return gate / (1 + torch.exp(-gate)) * up


_module = None


def _fp4():
    global _module
    if _module is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import ashqk

        _module = ashqk
    return _module


def run(state):
    op, fmt, dtype, g = state["op"], state["format"], state["dtype"], state["g"]
    if own:
        lib = _fp4()
        if op == "quantize":
            q = lib.quantize_fp4(state["x"], fmt, global_scale=g)
            return lib.dequantize_fp4(q, torch.bfloat16 if dtype == torch.float32 else dtype)
        if op == "gated":
            return lib.dequantize_fp4(lib.silu_mul_quantize_fp4(state["x"], fmt, global_scale=g), dtype)
        w = lib.FP4Tensor(*state["w"], (state["n"], state["k"]), fmt, state["wg"])
        if op == "matmul":
            return lib.fp4_matmul(lib.FP4Tensor(*state["a"], (state["m"], state["k"]), fmt, g), w, dtype)
        return lib.w4a4_linear(state["x"], w, global_scale=g, gated=op == "gated_linear")
    if op == "quantize":
        return _rounded(state["x"].float(), fmt, g).to(torch.bfloat16 if dtype == torch.float32 else dtype)
    if op == "gated":
        return _rounded(_silu_mul(state["x"]), fmt, g).to(dtype)
    w = _unpack(state["w"], fmt, state["wg"], state["k"])
    if op == "matmul":
        a = _unpack(state["a"], fmt, g, state["k"])
    else:
        a = _rounded(_silu_mul(state["x"]) if op == "gated_linear" else state["x"].float(), fmt, g)
    return (a @ w.t()).to(dtype)


# ---- the definition in 64 bits ----------------------------------------------------------------------


def _exact_rows(x, fmt, g):
    """64-bit rows as the format holds them: each magnitude's place among the midpoints of its neighbours."""
    rows, k = x.shape
    b = _BLOCK[fmt]
    out = torch.empty_like(x)
    for i in range(0, rows, 2048):
        part = x[i : i + 2048]
        pad = torch.nn.functional.pad(part, (0, -k % b)).unflatten(1, (-1, b))
        amax = pad.abs().amax(2, keepdim=True)
        if fmt == "mxfp4":
            s = torch.exp2(torch.floor(torch.log2(amax)).clamp(min=-125) - 2)
        else:
            s = (amax / 6 / g).clamp(max=448)
            unit = torch.exp2(torch.floor(torch.log2(s)).clamp(min=-6) - 3)  # E4M3's step at s
            s = torch.round(s / unit) * unit * g
        r = torch.where(s > 0, pad.abs() / s, 0.0)
        place = sum((r >= m).long() if up else (r > m).long() for m, up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)))
        v = torch.tensor(_VALUES, dtype=torch.float64, device=x.device)[place] * s
        out[i : i + 2048] = torch.where(pad < 0, -v, v).flatten(1)[:, :k]
    return out


def _exact_held(packed, fmt, g, k):
    codes, scales = (t.long() for t in packed)
    r = torch.arange(codes.shape[0], device=codes.device)[:, None]
    c = torch.arange(k, device=codes.device)[None]
    code = (codes[r, c // 2] >> (4 * (c % 2))) & 15
    b = c // _BLOCK[fmt]
    byte = scales[r // 128, b // 4, r % 32, r // 32 % 4, b % 4]
    exponent, mantissa = (code >> 1) & 3, code & 1
    v = torch.where(exponent > 0, (2 + mantissa).double() * torch.exp2(exponent.double() - 2), mantissa.double() / 2)
    v = torch.where(code > 7, -v, v)
    if fmt == "mxfp4":
        return v * torch.exp2(byte.double() - 127)
    e, m = byte >> 3, byte & 7
    return v * torch.where(e > 0, (8 + m).double() * torch.exp2(e.double() - 10), m.double() * 2.0**-9) * g


def exact(case, seed):
    state = prepare(case, seed)
    op, fmt, g, k = state["op"], state["format"], state["g"], state["k"]
    if op == "matmul":
        a = _exact_held(state["a"], fmt, g, k)
    else:
        x = state["x"].double()
        if op in ("gated", "gated_linear"):
            x = x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:]
        a = _exact_rows(x, fmt, g)
    if op in ("quantize", "gated"):
        return a
    return a @ _exact_held(state["w"], fmt, state["wg"], k).t()


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    op, m, k, fmt = case["op"], case["m"], case["k"], case["format"]
    size = 4 if case["dtype"] == "fp32" else 2
    held = 0.5 + 1 / _BLOCK[fmt]  # bytes of an element with its share of the scale
    if op in ("quantize", "gated"):
        # The rows read, the quantised form written and read back, 16-bit values written.
        read = m * k * size * (2 if op == "gated" else 1)
        return {"bytes": read + 2 * m * k * held + 2 * m * k, "flops": (8 if op == "gated" else 4) * m * k}
    n = case["n"]
    a = m * k * {"matmul": held, "linear": 2, "gated_linear": 4}[op]
    return {"bytes": a + n * k * held + 2 * m * n, "flops": 2 * m * n * k}
