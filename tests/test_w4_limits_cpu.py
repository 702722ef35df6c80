"""Weights that cannot be quantised, and packed weights that are not what they claim (no GPU)."""
import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import quantize_w4


@pytest.mark.parametrize("symmetric", [False, True])
def test_weights_that_are_not_finite_are_refused(symmetric):
    for value in (float("nan"), float("inf"), float("-inf")):
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            w = torch.randn(4, 64).to(dtype)
            w[2, 40] = value
            with pytest.raises(ValueError):
                quantize_w4(w, 32, symmetric=symmetric)
    with pytest.raises(ValueError):  # finite, but their scales are past fp16
        quantize_w4(torch.randn(4, 64) * 1e7, 32, symmetric=symmetric, dtype=torch.float16)
    for shape in ((4, 0), (0, 64)):
        with pytest.raises(ValueError):
            quantize_w4(torch.zeros(shape), 32, symmetric=symmetric)


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("size", [1e-33, 1e-20, 1.0, 1e30])
def test_small_and_large_weights_keep_their_relative_error(symmetric, size):
    """As for weights of ordinary size: half a step and the rounding of the scale to bf16, which moves a code's
    value by up to 15 (8) of its half steps of 2^-8, and a clamped end by as much again."""
    torch.manual_seed(1)
    w = torch.randn(6, 128) * size
    v = w.view(6, -1, 32)
    step = v.abs().amax(-1) / 7 if symmetric else (v.amax(-1).clamp_min(0) - v.amin(-1).clamp_max(0)) / 15
    off = (quantize_w4(w, 32, symmetric=symmetric).dequantize().view_as(v) - v).abs()
    assert (off <= step[..., None] * (1.0 + 16 * 2.0 ** -8)).all()
