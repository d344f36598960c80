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


def _two_layers():
    from ashqk.awq_checkpoint import AWQLayer

    layer = AWQLayer(torch.zeros(128, 4, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, 32, dtype=torch.float16), None)
    model = torch.nn.Sequential()
    for name in ("a", "b"):
        model.add_module(name, torch.nn.Linear(128, 32))
    return model, {"a": layer, "b": layer}


def test_input_scales_reach_the_layers(monkeypatch):
    from ashqk.awq_checkpoint import replace_linear_layers

    model, layers = _two_layers()
    seen = []
    monkeypatch.setattr(ashqk.FP4Linear, "from_awq", staticmethod(lambda layer, fmt, **kw: seen.append((fmt, kw)) or torch.nn.Identity()))
    assert replace_linear_layers(model, layers, "nvfp4", {"a": 0.25, "b": 0.5}) == ["a", "b"]
    assert seen == [("nvfp4", {"input_global_scale": 0.25}), ("nvfp4", {"input_global_scale": 0.5})]


@pytest.mark.parametrize("fmt,scales,error", [("nvfp4", {"a": 0.25}, KeyError), ("nvfp4", {"a": 1.0, "b": 1.0, "c": 1.0}, KeyError),
                                              ("nvfp4", {"a": 0.25, "b": 0.0}, ValueError), ("nvfp4", {"a": float("nan"), "b": 1.0}, ValueError),
                                              ("mxfp4", {"a": 1.0, "b": 1.0}, ValueError), (None, {"a": 1.0, "b": 1.0}, ValueError)])
def test_input_scales_that_do_not_fit_replace_nothing(fmt, scales, error):
    from ashqk.awq_checkpoint import replace_linear_layers

    model, layers = _two_layers()
    with pytest.raises(error):
        replace_linear_layers(model, layers, fmt, scales)
    assert all(type(m) is torch.nn.Linear for m in model)


def test_conversion_without_an_input_scale_warns(monkeypatch):
    w = ashqk.FP4Tensor(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), (8, 64), "nvfp4", 0.5)
    monkeypatch.setattr(ashqk.fp4, "quantize_fp4", lambda *a, **kw: w)
    with pytest.warns(UserWarning, match="input_global_scale"):
        assert ashqk.FP4Linear.from_float(torch.ones(8, 64)).input_global_scale == 1.0
    import warnings

    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert ashqk.FP4Linear.from_float(torch.ones(8, 64), input_global_scale=0.25).input_global_scale == 0.25


def test_negative_block_scales_are_refused():
    codes = torch.zeros(3, 32, dtype=torch.uint8)
    scales = torch.ones(3, 4)
    scales[2, 1] = -0.5
    for bad in (scales.to(torch.float8_e4m3fn), scales.to(torch.float8_e4m3fn).view(torch.uint8)):
        with pytest.raises(AssertionError, match="negative"):
            ashqk.FP4Tensor.from_rowmajor(codes, bad, "nvfp4")
    ashqk.FP4Tensor.from_rowmajor(codes, torch.full((3, 2), 200, dtype=torch.uint8), "mxfp4")  # E8M0 has no sign
    nan = torch.full((3, 4), 127, dtype=torch.uint8)
    assert int(ashqk.FP4Tensor.from_rowmajor(codes, nan, "nvfp4").scales_rowmajor().min()) == 127
    ashqk.FP4Tensor.from_rowmajor(codes[:0], nan[:0], "nvfp4")


def test_a_trained_layers_bias_brings_no_gradient():
    """``FP4Linear(w, linear.bias)``: the layer has no gradients, so its output must not ask for one and be refused by the
    next layer."""
    w = ashqk.FP4Tensor(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), (8, 64))
    linear = torch.nn.Linear(64, 8)
    layer = ashqk.FP4Linear(w, linear.bias)
    assert not layer.bias.requires_grad and type(layer.bias) is torch.Tensor and torch.equal(layer.bias, linear.bias)
    assert linear.bias.requires_grad
