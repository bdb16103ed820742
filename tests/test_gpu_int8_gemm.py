"""int8_gemm_nt against sums in 64 bits.

Tolerances: the sum is exact and rounded once to fp32, the two scales and C (or SwiGLU) add a rounding
each: value within 4 2^-24 of the sum of |scaled product| and |C|, then half a step of the type. SwiGLU:
gate and up within 3 2^-24 each; d silu / silu is at most 1 + |g| of dg / g, the sigmoid's exponential and
reciprocal are off by 2^-22 each with fast_math (hardware exp2 and reciprocal, 1 unit each, and the rounded
product g log2 e, |g| 2^-24), so (16 + 8 |g|) 2^-24 of the value covers both forms."""
import pytest
import torch

from tests.gpu_common import need_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = (torch.bfloat16, torch.float16, torch.float32)


def make(m, n, k, seed=0, full=False):
    torch.manual_seed(seed)
    if full:
        q = lambda r: torch.randint(-128, 128, (r, k), device="cuda", dtype=torch.int8)
    else:
        q = lambda r: (torch.randn((r, k), device="cuda") * 33).round().clamp(-127, 127).to(torch.int8)
    s = lambda r: torch.rand(r, device="cuda") * 0.02 + 0.001
    return (q(m), s(m)), (q(n), s(n))


def product(a, b):
    # (exact: |sums| < 2^53)
    return (a[0].double() @ b[0].double().t()) * a[1].double()[:, None] * b[1].double()


def check(d, ref, mag, c=4.0):
    fi = torch.finfo(d.dtype)
    tol = ref.abs() * (fi.eps / 2) + c * U * mag * (1 + fi.eps) + fi.tiny
    over = ref.abs() > fi.max
    bad = ~(((d.double() - ref).abs() <= tol) | (over & torch.isinf(d) & (d.double() * ref > 0)))
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())


def check_swiglu(d, ref, clamp):
    g, u = ref.chunk(2, 1)
    c = clamp if clamp is not None else float("inf")
    g, u = g.clamp(max=c), u.clamp(-c, c)
    want = g * torch.sigmoid(g) * u
    # (a sigmoid below the least normal number, g < -87, may be flushed to zero: off by 2^-126, times g u)
    check(d, want, want.abs() * (16 + 8 * g.abs()) + 2.0 ** -126 * (g * u).abs() / U, 1.0)


SHAPES = [(1, 1, 1), (1, 16, 64), (1, 4096, 2048), (2, 30, 16), (3, 7, 5), (5, 64, 48), (16, 16, 128), (17, 33, 80), (31, 100, 256),
          (33, 257, 112), (48, 512, 1024), (63, 130, 144), (64, 4096, 7168), (65, 128, 2048), (100, 384, 400), (128, 128, 128),
          (129, 320, 640), (200, 1000, 96), (255, 513, 272), (256, 256, 512), (300, 2880, 1024), (777, 640, 1296), (1000, 5120, 288),
          (2049, 1040, 160), (200, 1000, 512), (1000, 4000, 512), (2000, 4002, 528), (4000, 4000, 528), (3999, 4034, 400),
          (3, 10, 5), (20, 34, 21), (50, 66, 37), (300, 66, 129)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes(m, n, k):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = make(m, n, k, seed=m + n + k)
    ref = product(a, b)
    for dt in DT:
        d = torch.full((m, n), 7.0, dtype=dt, device="cuda")
        assert dgm.int8_gemm_nt(a, b, d) is d
        check(d, ref, ref.abs())
        c = torch.randn((m, n), device="cuda").to(dt)
        check(dgm.int8_gemm_nt(a, b, d, c=c), ref + c.double(), ref.abs() + c.double().abs())
        bias = torch.randn(n, device="cuda").to(dt)
        check(dgm.int8_gemm_nt(a, b, d, c=bias), ref + bias.double(), ref.abs() + bias.double().abs())
        d.copy_(c)
        check(dgm.int8_gemm_nt(a, b, d, c=d), ref + c.double(), ref.abs() + c.double().abs())
    if n % 2 == 0:
        for dt, clamp, fast in ((torch.bfloat16, 10.0, True), (torch.float32, 1.0, False), (torch.float16, None, True)):
            d = torch.full((m, n // 2), 7.0, dtype=dt, device="cuda")
            dgm.int8_gemm_nt(a, b, d, activation="swiglu", activation_clamp=clamp, fast_math=fast)
            check_swiglu(d, ref, clamp)


@pytest.mark.parametrize("m,n,k", [(1, 10, 2048), (1, 34, 4097), (2, 4098, 4112), (3, 2046, 2064), (5, 18, 7001), (7, 1030, 2192),
                                   (8, 2048, 4224), (8, 2050, 2064), (9, 2048, 2048), (2, 8206, 4109), (4, 8206, 4112),
                                   (16, 4090, 1040), (16, 4098, 1040), (31, 4096, 528), (50, 1026, 400)])
def test_few_tokens(m, n, k):
    """The forms that few tokens take: parts of K in a fragment, gate and up rows in one or two, edges in every direction."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for full in (False, True):
        a, b = make(m, n, k, seed=m + n + k, full=full)
        ref = product(a, b)
        f = torch.full((m + 1, n + 3), 7.0, device="cuda")
        check(dgm.int8_gemm_nt(a, b, f[:m, :n]), ref, ref.abs())
        assert bool((f[:, n:] == 7).all()) and bool((f[m:] == 7).all())
        c = torch.randn((m, n), device="cuda").to(torch.bfloat16)
        check(dgm.int8_gemm_nt(a, b, c.clone(), c=c), ref + c.double(), ref.abs() + c.double().abs())
        d = torch.full((m + 1, n // 2), 7.0, dtype=torch.bfloat16, device="cuda")
        check_swiglu(dgm.int8_gemm_nt(a, b, d[:m], activation="swiglu", activation_clamp=3.0), ref, 3.0)
        assert bool((d[m:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(69, 8278, 144), (200, 8242, 160), (392, 8206, 144), (586, 8292, 144), (4100, 1830, 144),
                                   (1025, 7226, 144), (1732, 6474, 144), (1543, 7174, 144), (50, 4246, 4112), (18, 7758, 4112),
                                   (65, 8270, 7184), (67, 4354, 7184), (133, 5502, 7184), (67, 8222, 10256), (135, 8284, 10256),
                                   (225, 8230, 10256), (585, 4106, 16400)])
def test_ragged_tiles(m, n, k):
    """The tile sizes that wide outputs and long sums take, whole and in ranges of K, with edges in every direction."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = make(m, n, k, seed=m + k)
    ref = product(a, b)
    d = torch.full((m + 1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    bias = torch.randn(n, device="cuda").to(torch.bfloat16)
    check(dgm.int8_gemm_nt(a, b, d[:m], c=bias), ref + bias.double(), ref.abs() + bias.double().abs())
    f = torch.full((m, n + 3), 7.0, device="cuda")
    check(dgm.int8_gemm_nt(a, b, f[:, :n]), ref, ref.abs())
    assert bool((d[m:] == 7).all()) and bool((f[:, n:] == 7).all())
    d = torch.full((m + 1, n // 2), 7.0, dtype=torch.bfloat16, device="cuda")
    check_swiglu(dgm.int8_gemm_nt(a, b, d[:m], activation="swiglu", activation_clamp=2.0), ref, 2.0)
    assert bool((d[m:] == 7).all())


@pytest.mark.parametrize("m", [1, 7, 40, 130, 400])
def test_extreme_values(m):
    """Codes over all of int8, -128 included; the largest k with every product 128 * 128; zero scales."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = make(m, 96, 1024, seed=m, full=True)
    a[1][0] = 0
    d = torch.empty((m, 96), dtype=torch.float32, device="cuda")
    ref = product(a, b)
    check(dgm.int8_gemm_nt(a, b, d), ref, ref.abs())
    assert not bool(d[0].any())
    K = 131071 // 16 * 16
    a = torch.full((m, K), -128, dtype=torch.int8, device="cuda"), torch.full((m,), 2.0 ** -20, device="cuda")
    b = torch.full((40, K), -128, dtype=torch.int8, device="cuda"), torch.full((40,), 2.0 ** -10, device="cuda")
    d = torch.empty((m, 40), dtype=torch.float32, device="cuda")
    want = torch.tensor(float(K * 16384), device="cuda") * 2.0 ** -30
    assert bool((dgm.int8_gemm_nt(a, b, d) == want).all())


def test_scales_as_the_cast_returns_them():
    """Rows and scales straight from per_token_cast_to_int8 and from rms_norm_residual."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    cast = dgm.quantization_qoq_fused.per_token_cast_to_int8
    torch.manual_seed(1)
    x, w = torch.randn((20, 512), device="cuda").bfloat16(), torch.randn((48, 512), device="cuda").bfloat16()
    a, b = cast(x), cast(w)
    assert a[1].shape == (20, 4)
    d = torch.empty((20, 48), dtype=torch.float32, device="cuda")
    ref = product((a[0], a[1][:, 0]), (b[0], b[1][:, 0]))
    check(dgm.int8_gemm_nt(a, b, d), ref, ref.abs())
    _, h, rows = dgm.rms_norm_residual(x, pre_weight=torch.ones(512, device="cuda").bfloat16(), quant="int8")
    ref = product(rows, (b[0], b[1][:, 0]))
    check(dgm.int8_gemm_nt(rows, b, d), ref, ref.abs())


@pytest.mark.parametrize("m", [3, 50, 300])
def test_strides_and_alignment(m):
    """Row strides, rows off 16-byte alignment, transposed operands, places in a wider d; nothing beside d's
    rows is written."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    n, k = 200, 320
    a, b = make(m, n, k, seed=m)
    ref = product(a, b)
    wide = lambda t, by, at: torch.full((t.size(0), t.size(1) + by), 9, dtype=t.dtype, device="cuda")[:, at:at + t.size(1)].copy_(t)
    for fa in (lambda t: wide(t, 16, 0), lambda t: wide(t, 16, 16), lambda t: wide(t, 5, 0), lambda t: wide(t, 32, 3),
               lambda t: t.t().contiguous().t()):
        for dt in (torch.bfloat16, torch.float32):
            for by, at in ((0, 0), (8, 8), (3, 1)):
                big = torch.full((m + 2, n + by), 5.0, dtype=dt, device="cuda")
                d = big[1:-1, at:at + n]
                check(dgm.int8_gemm_nt((fa(a[0]), a[1]), (fa(b[0]), b[1]), d), ref, ref.abs())
                rest = torch.ones_like(big, dtype=torch.bool)
                rest[1:-1, at:at + n] = False
                assert bool((big[rest] == 5).all())
    one = a[0][:1].expand(m, k)                         # the same token row for every token (stride 0)
    d = torch.empty((m, n), dtype=torch.float32, device="cuda")
    r = product((one, a[1]), b)
    check(dgm.int8_gemm_nt((one, a[1]), b, d), r, r.abs())
    every = torch.stack([a[1], a[1] * 3], 1)            # strided scales
    check(dgm.int8_gemm_nt((a[0], every[:, 0]), b, d), ref, ref.abs())
    cwide = torch.randn((m, n + 4), device="cuda")[:, 2:n + 2]
    check(dgm.int8_gemm_nt(a, b, d, c=cwide), ref + cwide.double(), ref.abs() + cwide.double().abs())
    bigd = torch.empty((m + 1, n), device="cuda")
    with pytest.raises(ValueError, match="c overlaps d"):
        dgm.int8_gemm_nt(a, b, bigd[:m], c=bigd[1:])
    raw = torch.zeros(m * k + m * n * 4, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError, match="d overlaps an operand"):
        dgm.int8_gemm_nt((raw[:m * k].view(m, k), a[1]), b, raw[m * k - 16:m * k - 16 + m * n * 2].view(torch.bfloat16).view(m, n))
    dgm.int8_gemm_nt((a[0][:0], a[1][:0]), b, d[:0])
    dgm.int8_gemm_nt(a, (b[0][:0], b[1][:0]), d[:, :0])


def test_rows_of_another_call_do_not_matter():
    """A token's results are the same bits whatever other tokens are in the call within one kernel's range,
    and for any number of tokens (sums are exact)."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = make(300, 192, 528, seed=4)
    full = torch.empty((300, 192), dtype=torch.float32, device="cuda")
    dgm.int8_gemm_nt(a, b, full)
    for m in (1, 16, 33, 64, 65, 129, 200):
        d = torch.empty((m, 192), dtype=torch.float32, device="cuda")
        dgm.int8_gemm_nt((a[0][:m], a[1][:m]), b, d)
        assert torch.equal(d, full[:m]), m


@pytest.mark.parametrize("m", [3, 70])
def test_offsets_beyond_32_bits(m):
    """Rows of every operand more than 2^31 bytes from the first one, in the register and the tile kernels."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    n, k = 48, 256
    a, b = make(m, n, k, seed=m)
    d = torch.empty((m, n), dtype=torch.float32, device="cuda")
    dgm.int8_gemm_nt(a, b, d)
    far = {}
    for name, rows, width, dt in (("a", m, k, torch.int8), ("b", n, k, torch.int8), ("d", m, n, torch.float32)):
        gap = (5 << 30) // rows // dt.itemsize // 16 * 16
        big = torch.empty(gap * (rows - 1) + width, dtype=dt, device="cuda")
        far[name] = big.as_strided((rows, width), (gap, 1))
    far["a"].copy_(a[0]), far["b"].copy_(b[0])
    dgm.int8_gemm_nt((far["a"], a[1]), (far["b"], b[1]), far["d"])
    assert torch.equal(far["d"], d)
    dgm.int8_gemm_nt((far["a"], a[1]), (far["b"], b[1]), far["d"], c=far["d"])
    assert torch.equal(far["d"], d + d)


def test_streams_and_graph():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for m in (2, 40, 150, 600):
        a, b = make(m, 1024, 2048, seed=m)
        d = torch.empty((m, 1024), dtype=torch.bfloat16, device="cuda")
        dgm.int8_gemm_nt(a, b, d)
        want = d.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        d2 = torch.empty_like(d)
        with torch.cuda.stream(side):
            dgm.int8_gemm_nt(a, b, d2)
        dgm.int8_gemm_nt(a, b, d)                        # two calls at once
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(d, want) and torch.equal(d2, want)
        graphs = []
        for out in (d, d2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                dgm.int8_gemm_nt(a, b, out)
            graphs.append(g)
        for i in range(3):
            a[0].copy_(torch.randint(-127, 128, a[0].shape, device="cuda", dtype=torch.int8))
            d.zero_(), d2.zero_()
            graphs[0].replay(), graphs[1].replay()
            torch.cuda.synchronize()
            eager = torch.empty_like(d)
            dgm.int8_gemm_nt(a, b, eager)
            assert torch.equal(d, eager) and torch.equal(d2, eager), (m, i)
