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
