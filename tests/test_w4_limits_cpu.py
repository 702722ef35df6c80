"""Weights that cannot be quantised, and packed weights that are not what they claim (no GPU)."""
import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import W4Weight, quantize_w4


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


def test_packed_weights_of_other_sizes_are_refused():
    """A W4Weight put together by hand, as a loader or a move to another device does."""
    w = quantize_w4(torch.randn(40, 320), 64)
    again = W4Weight(w.packed.clone(), w.n, w.k, w.group_size, w.dtype)
    assert torch.equal(again.dequantize(), w.dequantize())
    for packed in (w.packed[:-1], w.packed[16:], torch.cat([w.packed, w.packed]), w.packed.repeat_interleave(2)[::2]):
        with pytest.raises(ValueError):
            W4Weight(packed, w.n, w.k, w.group_size, w.dtype)
    for n, k, group in ((49, 320, 64), (40, 448, 64), (40, 320, 32), (40, 320, 128), (0, 320, 64), (40, 0, 64),
                        (40, 320, 16)):
        with pytest.raises(ValueError):
            W4Weight(w.packed, n, k, group, w.dtype)
    for packed, dtype in ((w.packed.float(), w.dtype), (None, w.dtype), (w.packed, torch.float32)):
        with pytest.raises(TypeError):
            W4Weight(packed, w.n, w.k, w.group_size, dtype)
