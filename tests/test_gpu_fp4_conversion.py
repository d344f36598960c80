"""AWQ layers converted to NVFP4, with activations far from 1."""

from __future__ import annotations

import pytest
import torch

import ashqk
from ashqk.awq_checkpoint import AWQLayer, replace_linear_layers
from oracle import awq_oracle as O
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e-3, 4e-3, 1.0, 3e3])
def test_input_scales_keep_activations_of_any_size(size):
    """Rows of N(0, size): with the scale of inputs like them, quantising moves each value by at most half a step of its
    element and its block's scale by at most half a step of E4M3, as for rows of N(0, 1)."""
    n, k = 384, 512
    _, qw, qz, s = O.make_problem(1, n, k, 128, seed=1)
    layer = AWQLayer(*(torch.from_numpy(t).cuda() for t in (qw, qz, s)), None)
    g = torch.Generator(device="cuda").manual_seed(3)
    seen, x = (torch.randn(m, k, generator=g, device="cuda", dtype=torch.float32) * size for m in (64, 20))
    x = x.clamp(seen.min(), seen.max()).bfloat16()
    model = torch.nn.Sequential()
    model.add_module("up", torch.nn.Linear(k, n, bias=False))
    gx = ashqk.fp4_global_scale(seen)
    replace_linear_layers(model, {"up": layer}, "nvfp4", {"up": gx})
    assert model.up.input_global_scale == gx
    y = model(x)
    # The product of what the oracle rounds x to, in 64 bits. fp32 sums: (K + 16) 2^-23 of the terms' magnitudes, the
    # scales' product one rounding more; then half a step of bf16.
    x64 = x.double().cpu().numpy()
    a = torch.from_numpy(F.values(*F.quantize(x64, "nvfp4", gx), "nvfp4", gx)).cuda()
    w = ashqk.dequantize_fp4(ashqk.FP4Tensor(model.up.codes, model.up.scales, (n, k), "nvfp4")).double() * model.up.global_scale
    want, terms = a @ w.t(), a.abs() @ w.abs().t()
    eps = torch.finfo(torch.bfloat16).eps / 2
    assert bool(((y.double() - want).abs() <= eps * want.abs() + (k + 17) * 2.0**-23 * terms * (1 + eps)).all())
    # And x itself is there: an element is off by at most a fifth of itself (5 between 4 and 6) or a quarter of its scale,
    # which is amax / 6 to within a sixteenth and can cut that much off the block's largest value.
    xd = torch.from_numpy(x64).cuda()
    amax = xd.abs().unflatten(1, (-1, 16)).amax(2).repeat_interleave(16, 1)
    bound = torch.maximum(xd.abs() / 5, amax / 6 / 4 * (1 + 2.0**-4)) + amax / 16
    assert bool(((a - xd).abs() <= bound * (1 + 2.0**-10)).all())


def test_layers_of_a_trained_model_in_a_row():
    """Linear layers with their own weights and biases, converted as they are and called outside no_grad."""
    torch.manual_seed(2)
    up, down = (torch.nn.Linear(128, 96).cuda().half(), torch.nn.Linear(96, 64).cuda().half())
    layers = [ashqk.FP4Linear.from_float(m.weight, m.bias, "mxfp4") for m in (up, down)]
    x = torch.randn(5, 128, device="cuda", dtype=torch.float16)
    h = layers[0](x)
    y = layers[1](h)
    assert not y.requires_grad
    assert torch.equal(h, ashqk.w4a4_linear(x, ashqk.quantize_fp4(up.weight.detach())) + up.bias.detach())
    assert torch.equal(y, ashqk.w4a4_linear(h, ashqk.quantize_fp4(down.weight.detach())) + down.bias.detach())
