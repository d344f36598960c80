"""Stream order across launches that overlap (programmatic dependent launch), read from the kernels' sources.

A grid that lets its dependents start before its own ``griddepcontrol.wait`` has returned lets them start while the
launch before it still writes. The decode GEMVs load their weights before they wait, so behind such a grid they could
read weights that are still being written. Every 4-bit floating-point kernel must wait first.
"""

from __future__ import annotations

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ash-quant-kernels_b200", "csrc")
SOURCES = sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "fp4_*.cu")))


def _kernels(text):
    """The bodies of the __global__ functions."""
    for m in re.finditer(r"__global__", text):
        start = text.index("{", m.end())
        depth = 0
        for i in range(start, len(text)):
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            if depth == 0:
                yield text[start:i]
                break


@pytest.mark.parametrize("source", SOURCES)
def test_dependents_start_behind_the_wait(source):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, source)).read())
    for body in _kernels(text):
        assert body.count("pdl_wait();") == 1
        before = body[: body.index("pdl_wait();")]
        assert "pdl_launch_dependents" not in before, "dependents are let go before the wait"
        # what runs ahead of the wait may fetch into L2, which is coherent, but neither load nor store
        for word in ("tma_load", "bulk_load", "ld_once", "load16", "quantize_slice", "store4("):
            assert word not in before, word


def test_every_kernel_is_looked_at():
    found = {s: len(list(_kernels(open(os.path.join(CSRC, s)).read()))) for s in SOURCES}
    assert found == {"fp4_gemm_pair.cu": 1, "fp4_gemm_rows.cu": 1, "fp4_linear.cu": 0, "fp4_quant.cu": 3}
