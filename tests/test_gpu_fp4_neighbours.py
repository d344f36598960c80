"""4-bit floating-point products among launches of other kernels, on their own stream and on others."""

from __future__ import annotations

import pytest
import torch

import ashqk
from oracle import awq_oracle as O

pytestmark = pytest.mark.gpu


def operands(m, n, k, fmt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    w = torch.randn(n, k, generator=g, device="cuda", dtype=torch.float32) * 0.02
    return x, ashqk.quantize_fp4(w, fmt, global_scale=1 / 1024 if fmt == "nvfp4" else 1.0)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [17, 20, 32, 40, 64, 100, 128])
@pytest.mark.parametrize("n", [512, 4096])
def test_products_between_decode_calls(fmt, m, n):
    """Sums that travel between CTAs in bulk copies, with decode GEMVs (whose first loads go to shared memory as soon as
    a CTA fits) right behind them and beside them: the same bits as alone."""
    x, w = operands(m, n, 4096, fmt, m + n)
    q = ashqk.quantize_fp4(x, fmt)
    xa, qw, qz, s = (torch.from_numpy(t).cuda() for t in O.make_problem(1, 2048, 4096, 128, seed=m))
    jobs = [lambda: ashqk.w4a4_linear(x, w), lambda: ashqk.fp4_matmul(q, w), lambda: ashqk.w4a16_linear(xa, qw, qz, s)]
    want = []
    for job in jobs:
        want.append(job())
        torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    for st in side:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        for i, job in enumerate(jobs):
            got.append((i, job()))
            got.append((2, jobs[2]()))
        for st in side:
            with torch.cuda.stream(st):
                got += [(2, jobs[2]()) for _ in range(3)]
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i]), i


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [1, 16, 32, 100, 300])
@pytest.mark.parametrize("call", ["linear", "matmul", "gated", "quantize", "dequantize"])
def test_awq_weights_written_before_a_call(fmt, m, call):
    """AWQ weights written, a 4-bit floating-point call, a decode GEMV on those weights: no wait in between, and the GEMV
    multiplies what was written."""
    x, w = operands(m, 512, 1024, fmt, m)
    q = ashqk.quantize_fp4(x, fmt)
    x2 = x.repeat(1, 2)
    between = {"linear": lambda: ashqk.w4a4_linear(x, w), "matmul": lambda: ashqk.fp4_matmul(q, w), "gated": lambda: ashqk.w4a4_linear(x2, w, gated=True),
               "quantize": lambda: ashqk.quantize_fp4(x, fmt), "dequantize": lambda: ashqk.dequantize_fp4(q)}[call]
    problems = [[torch.from_numpy(t).cuda() for t in O.make_problem(1, 16384, 4096, 128, seed=s)] for s in range(2)]
    xa = problems[0][0]
    want = [ashqk.w4a16_linear(xa, *p[1:]) for p in problems]
    between()
    qw, qz, s = (torch.empty_like(t) for t in problems[0][1:])
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        _, nqw, nqz, ns = problems[i % 2]
        qz.copy_(nqz)
        s.copy_(ns)
        qw.copy_(nqw)
        between()
        got.append(ashqk.w4a16_linear(xa, qw, qz, s))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2]), i
