"""4-bit linear against its definition in 64 bits (GPU)."""
import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import _native, pack_w4, quantize_w4, w4_linear

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def weight(n, k, group, dtype, zeros=True, seed=0, lo=0, hi=15):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(lo, hi + 1, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    s = (0.004 + 0.008 * torch.rand(n, k // group, generator=g, device="cuda")).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return q, s, z


def activations(m, k, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    x[:, ::53] *= 10.0
    return x.to(dtype)


def check(y, x, q, s, z, residual=None):
    """|y - ref| within the output's rounding plus the fp32 sums' worst case, and the norm of the
    whole within the output's rounding alone.

    Inside a group of g inputs the integers off + q (off = 256 or 16) are summed by g/16 mma steps, each
    off by at most 2 units of 2^-23 of the magnitude summed; offset and zero point are two more
    roundings (A below bounds all of these magnitudes). The scaled groups are then added in at most
    K/g + 72 roundings (slices of up to 8 warps and 8 CTAs, residual) relative to sum |x w| and the
    residual (B). bf16 activations in fp16 are exact but for 2^-39 of the greatest of 128: covered by B.
    """
    n, k = q.shape
    g = k // s.shape[1]
    rep = lambda t: t.repeat_interleave(g, dim=1).double()  # noqa: E731
    zz = 8.0 if z is None else rep(z)
    w = (q.double() - zz) * rep(s)
    xd = x.double()
    ref = xd @ w.t()
    a = xd.abs() @ ((512.0 + q.double() + zz) * rep(s)).t()
    b = xd.abs() @ w.abs().t()
    if residual is not None:
        ref = ref + residual.double()
        b = b + residual.double().abs()
    half_step = torch.finfo(y.dtype).eps / 2
    tol = half_step * ref.abs() + 2.0 ** -23 * ((g / 8 + 2) * a + (k / g + 72) * b) + torch.finfo(y.dtype).tiny
    err = (y.double() - ref).abs()
    assert torch.isfinite(y).all()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3g} of the tolerance"
    assert err.norm() <= half_step * ref.norm() + 2.0 ** -23 * (a.norm() + b.norm())


SHAPES = [(1, 16, 128), (1, 1, 32), (2, 5, 96), (8, 100, 160), (9, 333, 4096), (16, 1000, 256), (17, 64, 512),
          (33, 48, 1024), (64, 130, 2048), (65, 70, 640), (130, 33, 128), (3, 40, 14336), (1, 6144, 4096),
          (40, 200, 14336), (7, 4100, 2080)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matches_definition(m, n, k, dtype):
    for group in (32, 64, 128):
        if k % group:
            continue
        q, s, z = weight(n, k, group, dtype, zeros=(m + group) % 3 != 0, seed=m + n + group)
        x = activations(m, k, dtype)
        y = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        got = w4_linear(x, pack_w4(q, s, z), y)
        assert got is y
        check(y, x, q, s, z)
    assert _native.device_error() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m", [1, 5, 20, 70])
def test_residual_may_be_the_output(m, dtype):
    q, s, z = weight(210, 512, 64, dtype)
    x, r = activations(m, 512, dtype), activations(m, 210, dtype, seed=3)
    w = pack_w4(q, s, z)
    check(w4_linear(x, w, residual=r), x, q, s, z, r)
    y = r.clone()
    w4_linear(x, w, y, residual=y)
    check(y, x, q, s, z, r)


@pytest.mark.parametrize("codes,zero", [((0, 0), 15), ((15, 15), 0), ((0, 0), 0), ((15, 15), 15)])
def test_extreme_codes(codes, zero):
    q, s, _ = weight(64, 256, 32, BF16, lo=codes[0], hi=codes[1])
    z = torch.full((64, 8), zero, dtype=torch.uint8, device="cuda")
    x = activations(4, 256, BF16)
    y = w4_linear(x, pack_w4(q, s, z))
    check(y, x, q, s, z)
    if codes[0] == zero:  # every weight is 0: so is the result, up to the sums' rounding checked above
        assert y.abs().max().item() < 1e-2


def test_strided_rows_streams_and_repeats():
    q, s, z = weight(300, 1024, 128, BF16)
    w = pack_w4(q, s, z)
    wide = activations(6, 1024 + 512, BF16)
    x = wide[:, 256:1280]
    y = w4_linear(x, w)
    check(y, x, q, s, z)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    y2 = torch.empty_like(y)
    w4_linear(x, w, y2, stream=st)
    st.synchronize()
    assert torch.equal(y, y2)
    for _ in range(20):
        assert torch.equal(w4_linear(x, w), y)


def test_zero_tokens_and_graph_replay():
    q, s, z = weight(96, 640, 128, FP16)
    w = pack_w4(q, s, z)
    assert w4_linear(torch.empty(0, 640, dtype=FP16, device="cuda"), w).shape == (0, 96)
    x, y = activations(3, 640, FP16), torch.empty(3, 96, dtype=FP16, device="cuda")
    w4_linear(x, w, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w4_linear(x, w, y)
        w4_linear(x, w, y, residual=y)  # y = 2 x W^T, rounded twice
    for seed in (5, 6):
        x.copy_(activations(3, 640, FP16, seed=seed))
        graph.replay()
        one = w4_linear(x, w)
        two = w4_linear(x, w, residual=one)
        assert torch.equal(y, two)


def test_quantized_weight_times_tokens():
    torch.manual_seed(0)
    for symmetric in (False, True):
        w = torch.randn(200, 384, device="cuda") * 0.02
        p = quantize_w4(w, 64, symmetric=symmetric)
        x = activations(4, 384, BF16)
        # The codes' half step (asymmetric: range / 15, symmetric: max / 7), with the scale's own rounding to
        # bf16 moving a code's value by up to 15 (8) of its half steps of 2^-8.
        v = w.view(200, -1, 64)
        step = (v.amax(-1).clamp_min(0) - v.amin(-1).clamp_max(0)) / 15 if not symmetric else v.abs().amax(-1) / 7
        off = (p.dequantize().view(200, -1, 64) - v).abs()
        assert (off <= step[..., None] * (1.0 + 16 * 2.0 ** -8)).all()
        y = w4_linear(x, p).double()
        ref = x.double() @ p.dequantize().double().t()
        assert ((y - ref).norm() / ref.norm()).item() <= 2.0 ** -8


def test_refusals():
    q, s, z = weight(32, 256, 64, BF16)
    w = pack_w4(q, s, z)
    x = activations(2, 256, BF16)
    with pytest.raises(TypeError):
        w4_linear(x.half(), w)
    with pytest.raises(TypeError):
        w4_linear(x, q)
    with pytest.raises(ValueError):
        w4_linear(x[:, :192], w)
    with pytest.raises(ValueError):
        w4_linear(x.t().contiguous().t(), w)  # columns are not dense
    with pytest.raises(ValueError):
        w4_linear(activations(2, 260, BF16)[:, :256], w)  # row stride 260
    with pytest.raises(ValueError):
        w4_linear(x, w, torch.empty(2, 33, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError):
        w4_linear(x, w, residual=torch.empty(1, 32, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError):  # 2-byte aligned rows
        w4_linear(torch.empty(2 * 256 + 1, dtype=BF16, device="cuda")[1:].view(2, 256), w)


# Sizes that take the ways the shapes above do not: output rows in several rounds per cluster (with a
# last slab of one block), inputs staged in several pieces, one row tile for a whole cluster, many
# passes of tokens, one block of inputs.
@pytest.mark.parametrize("m,n,k,group", [(16, 70000, 800, 32), (9, 70000, 896, 128), (16, 40, 20480, 64),
                                         (10, 700, 20480, 32), (64, 16400, 512, 128), (130, 6200, 640, 64),
                                         (70, 210, 512, 32), (50, 128, 14336, 128), (1000, 48, 256, 64),
                                         (17, 1, 32, 32), (64, 20000, 1152, 32), (40, 70000, 896, 32),
                                         (200, 30000, 128, 128), (33, 25000, 640, 64)])
def test_splits_and_rounds(m, n, k, group):
    q, s, z = weight(n, k, group, BF16, seed=n)
    x = activations(m, k, BF16)
    y = torch.full((m, n), float("nan"), dtype=BF16, device="cuda")
    w4_linear(x, pack_w4(q, s, z), y)
    check(y, x, q, s, z)
    assert _native.device_error() == 0


@pytest.mark.parametrize("m", [4, 40])
def test_two_streams_at_once_and_strided_rows(m):
    q, s, z = weight(1000, 2048, 64, BF16, seed=m)
    w = pack_w4(q, s, z)
    xs = [activations(m, 2048 + 1024, BF16, seed=i)[:, 512:2560] for i in range(2)]
    want = [w4_linear(x, w) for x in xs]
    for x, y in zip(xs, want):
        check(y, x, q, s, z)
    streams = [torch.cuda.Stream() for _ in xs]
    outs = [torch.zeros(20, m, 1000, dtype=BF16, device="cuda") for _ in xs]
    torch.cuda.synchronize()
    for i in range(20):
        for x, o, st in zip(xs, outs, streams):
            w4_linear(x, w, o[i], stream=st)
    torch.cuda.synchronize()
    for o, y in zip(outs, want):
        assert all(torch.equal(o[i], y) for i in range(20))


def test_infinite_and_nan_activations_stay_in_their_rows():
    for m in (3, 33):
        q, s, z = weight(130, 512, 64, BF16)
        w = pack_w4(q, s, z)
        x = activations(m, 512, BF16)
        clean = w4_linear(x, w)
        x[1, 100], x[2, 7] = float("nan"), float("inf")
        y = w4_linear(x, w)
        rest = [i for i in range(m) if i not in (1, 2)]
        assert torch.equal(y[rest], clean[rest])
        assert y[1].isnan().all() and not y[2].isfinite().any()


def test_overlaps_are_refused():
    q, s, z = weight(256, 256, 64, BF16)
    w = pack_w4(q, s, z)
    for m in (2, 20):
        buf = torch.zeros(4 * m, 256, dtype=BF16, device="cuda")
        x = buf[:m]
        for out in (x, buf[m - 1:2 * m - 1]):
            with pytest.raises(ValueError):
                w4_linear(x, w, out)
        with pytest.raises(ValueError):
            w4_linear(x, w, buf[m:2 * m], residual=buf[m + 1:2 * m + 1])
        w4_linear(x, w, buf[m:2 * m], residual=buf[2 * m:3 * m])


def test_captured_chain_of_layers():
    """Two layers, the second on the first one's output, and a residual onto it, replayed on new inputs."""
    for m in (12, 40, 100):
        q1, s1, z1 = weight(512, 384, 64, BF16, seed=1)
        q2, s2, z2 = weight(384, 512, 128, BF16, seed=2)
        w1, w2 = pack_w4(q1, s1, z1), pack_w4(q2, s2, z2)
        x = activations(m, 384, BF16)
        h = torch.empty(m, 512, dtype=BF16, device="cuda")
        y = torch.empty(m, 384, dtype=BF16, device="cuda")

        def step():
            w4_linear(x, w1, h)
            w4_linear(h, w2, y, residual=x)
            w4_linear(y, w1, h, residual=h)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(3):
                step()
        for seed in (7, 8):
            x.copy_(activations(m, 384, BF16, seed=seed))
            graph.replay()
            first = w4_linear(x, w1)
            check(first, x, q1, s1, z1)
            mid = w4_linear(first, w2, residual=x)
            check(mid, first, q2, s2, z2, x)
            assert torch.equal(y, mid)
            assert torch.equal(h, w4_linear(mid, w1, residual=first))
