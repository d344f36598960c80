"""Scales that callers choose or bring along, without a GPU."""

from __future__ import annotations

import pytest
import torch

import ashqk
from oracle import fp4_oracle as F


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("amax", [1e-38, 1e-19, 1e-16, 2.6e-15, 2.8e-15, 1e-3, 1.0, 5e4, 2.6e21])
def test_global_scale_of_any_tensor_is_one_that_the_quantiser_takes(amax, dtype):
    x = torch.tensor([[amax] + [amax / 7] * 15, [-amax / 2] * 16], dtype=dtype)
    g = ashqk.fp4_global_scale(x)
    ashqk.fp4._check("nvfp4", g)
    code, byte = F.quantize(x.double().numpy(), "nvfp4", g)
    if amax > 6 * 2.0**-9 * 1e-18:  # the smallest scale that the format has
        assert byte[:, 0].all() and code[0, 0] and code[1, 0], "a nonzero tensor became zeros"
    if amax >= 2.7e-15:
        assert g == pytest.approx(float(x.abs().max()) / 2688, rel=2.0**-23)


def test_global_scale_refuses_what_no_scale_holds():
    for amax in (2.8e21, 3e38):
        with pytest.raises(AssertionError, match="beyond"):
            ashqk.fp4_global_scale(torch.tensor([0.0, -amax]))
    assert ashqk.fp4_global_scale(torch.zeros(3, dtype=torch.float16)) == 1.0
