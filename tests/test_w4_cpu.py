"""The 4-bit weight's layout and the refusals that need no GPU."""
import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import W4Weight, _native, pack_w4, quantize_w4, w4_linear


@pytest.mark.parametrize("n,k,group,zeros,dtype", [
    (5, 32, 32, True, torch.bfloat16), (16, 128, 128, False, torch.float16), (37, 320, 64, True, torch.float16),
    (100, 4000, 32, False, torch.bfloat16), (1, 128, 64, True, torch.bfloat16)])
def test_pack_and_dequantize(n, k, group, zeros, dtype):
    torch.manual_seed(n)
    q = torch.randint(0, 16, (n, k), dtype=torch.uint8)
    s = torch.rand(n, k // group).to(dtype)
    z = torch.randint(0, 16, (n, k // group), dtype=torch.uint8) if zeros else None
    w = pack_w4(q, s, z)
    zz = 8.0 if z is None else z.float().repeat_interleave(group, 1)
    assert torch.equal(w.dequantize(), (q.float() - zz) * s.float().repeat_interleave(group, 1))
    # Where one element of the weight lies, by the layout's definition.
    row, col = n - 1, k - 1
    h, g = (row % 16) // 8, row % 8
    j, c, i = (col % 128) // 32, (col % 32) // 8, col % 8
    nb, kb, words = -(-n // 16), -(-k // 128), 256 + 2048 // group
    slab, block = col // 256, col % 256 // 128
    at = (slab * 2 * nb + (row // 16) * min(2, kb - 2 * slab) + block) * words
    word = int(w.packed[at + (h * 32 + 4 * g + c) * 4 + j]) & 0xFFFFFFFF
    word = (word >> 2) | (word & 3) << 30
    nibble = (i % 2) * 4 + i // 2  # even inputs in the low half, odd ones in the high half
    assert (word >> (4 * nibble)) & 15 == int(q[row, col])


def test_quantize_keeps_exact_grids():
    """A weight that is already (q - z) s with the full range of codes comes back exactly."""
    torch.manual_seed(0)
    q = torch.randint(0, 16, (12, 128), dtype=torch.uint8)
    q[:, 0::32], q[:, 1::32] = 0, 15
    w = (q.float() - 6.0) * 0.25
    assert torch.equal(quantize_w4(w, 32).dequantize(), w)
    assert torch.equal(quantize_w4(torch.zeros(3, 64), 32).dequantize(), torch.zeros(3, 64))


def test_refusals():
    q, s = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 2, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        pack_w4(q.int(), s)
    with pytest.raises(TypeError):
        pack_w4(q, s.float())
    with pytest.raises(TypeError):
        pack_w4(q, s, q.int())
    with pytest.raises(ValueError):
        pack_w4(q, s[:3])
    with pytest.raises(ValueError):
        pack_w4(q, torch.ones(4, 4, dtype=torch.bfloat16))  # groups of 16
    with pytest.raises(ValueError):
        pack_w4(q + 16, s)
    with pytest.raises(ValueError):
        pack_w4(q, s, torch.full((4, 2), 16, dtype=torch.uint8))
    with pytest.raises(ValueError):
        pack_w4(q, s, torch.zeros(4, 1, dtype=torch.uint8))
    with pytest.raises(ValueError):
        quantize_w4(torch.zeros(4, 100), 64)
    with pytest.raises(ValueError):  # CPU tensors
        w4_linear(torch.zeros(1, 64, dtype=torch.bfloat16), pack_w4(q, s))
    assert isinstance(pack_w4(q, s), W4Weight)


def test_entry_point_refuses_before_launch():
    lib = _native.load()

    def call(ldx=256, x=16, dtype=0, m=1, n=16, k=256, group=64):
        return lib.fk_w4_linear(x, ldx, 16, None, 16, dtype, m, n, k, group, None)

    for bad in (dict(ldx=255), dict(ldx=264 - 4), dict(x=18), dict(x=None), dict(dtype=2), dict(m=0), dict(n=0),
                dict(k=0), dict(group=16), dict(k=224)):
        assert call(**bad) == -1, bad
        assert lib.fk_last_error()


def test_entry_point_refuses_overlaps():
    lib = _native.load()

    def call(x=1 << 20, packed=1 << 24, residual=None, y=1 << 28):  # addresses are compared, never read
        return lib.fk_w4_linear(x, 512, packed, residual, y, 0, 3, 100, 256, 64, None)

    y = 1 << 28
    x_bytes, w_bytes, y_bytes = 2 * (2 * 512 + 256), 7 * 2 * (1024 + 128), 2 * 3 * 100
    for bad in (dict(x=y), dict(x=y - x_bytes + 16), dict(x=y + y_bytes - 8), dict(packed=y - w_bytes + 16),
                dict(packed=y + 592), dict(residual=y + 2), dict(residual=y - 2)):
        assert call(**bad) == -1, bad
        assert b"overlap" in lib.fk_last_error() or b"other memory" in lib.fk_last_error()
