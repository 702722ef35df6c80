"""The 4-bit linear around the sizes at which its two forms change places (GPU)."""
import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import _native, pack_w4, w4_linear
from test_w4_gpu import activations, check, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [8, 9, 16, 17])
@pytest.mark.parametrize("tiles", [1.0, 1.6, 2.0, 2.2, 2.6])
def test_borders(tiles, m, group, dtype):
    """One row below and above so many tiles of 128 rows per SM."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for n in (int(tiles * sms) * 128, int(tiles * sms) * 128 + 1):
        q, s, z = weight(n, 384, group, dtype, seed=n)
        x = activations(m, 384, dtype)
        y = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        w4_linear(x, pack_w4(q, s, z), y)
        check(y, x, q, s, z)
    assert _native.device_error() == 0
