"""mxfp4_quantize, mxfp4_gemm_nt and mxfp4_linear against their definitions in 64 bits.

Codes and scales are equal or wrong. Products: each product of two codes is exact; an instruction adds 128 of them, a
wave K / 128 instructions' sums, and up to 8 waves' and 8 ranges' sums are added to that. However an instruction adds,
a term passes at most 128 + K / 128 + 16 additions of fp32 numbers, each off by 2^-23 of its sum at most (2^-24 where
they round to nearest), and C one more: value within (145 + K / 128) 2^-23 of the sum of |products| and |C|, then half
a step of the type. SwiGLU: the above times (1 + |g|) for the gate's share, and (16 + 8 |g|) 2^-24 of the value as for
int8_gemm_nt. Where all sums are whole numbers of quarters below 2^24 they have to be exact."""
import pytest
import torch

from tests.gpu_common import need_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = (torch.bfloat16, torch.float16, torch.float32)
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def power(e):
    """2^e as fp64, by its bits"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantized(x, floor=1e-30):
    """(codes, scales) of x's rows by the definition, in 64 bits."""
    t = x.double()
    t = torch.cat([t, t.new_zeros(t.size(0), -t.size(1) % 32)], 1).reshape(t.size(0), -1, 32)
    bad = ~torch.isfinite(t).all(2)
    t = torch.where(bad[:, :, None], torch.zeros_like(t), t)
    floor = float(torch.tensor(floor, dtype=torch.float32))
    mantissa, exponent = torch.frexp(t.abs().amax(2).clamp(min=floor) / 6)
    e = torch.where(mantissa == 0, torch.full_like(exponent, -126), exponent - (mantissa == 0.5).int()).clamp(-126, 127)
    y = t / power(e)[:, :, None]
    index = sum((y.abs() > mid).int() for mid in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
    code = (index + 8 * ((y < 0) & (index > 0)).int()).flatten(1).to(torch.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def values(pair):
    codes, scales = pair
    code = torch.stack([codes & 15, codes >> 4], 2).flatten(1).long()
    v = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=codes.device)[code]
    s = torch.where(scales == 255, torch.full_like(scales, 0, dtype=torch.float64) + float("nan"), power(scales.int() - 127))
    return (v.reshape(v.size(0), -1, 32) * s[:, :, None]).flatten(1)


def same(got, want):
    assert got[0].dtype == got[1].dtype == torch.uint8
    assert got[0].shape == want[0].shape and got[1].shape == want[1].shape, (got[0].shape, want[0].shape)
    assert torch.equal(got[1], want[1]), torch.nonzero(got[1] != want[1])[:4].tolist()
    assert torch.equal(got[0], want[0]), torch.nonzero(got[0] != want[0])[:4].tolist()


def rows(m, k, dtype, seed=0):
    """Values of every size, midpoints between codes and exact multiples of 6 among them, both zeros."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    x = rnd(m, k) * torch.exp2(torch.randint(-9, 9, (m, k), generator=g, device="cuda").float() * (rnd(m, 1) > 0))
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0], device="cuda")
    pick = mids[torch.randint(0, 9, (m, k), generator=g, device="cuda")] * torch.where(rnd(m, k) > 0, 1.0, -1.0)
    scale = torch.exp2(torch.randint(-6, 6, (m, 1), generator=g, device="cuda").float())
    return torch.where(rnd(m, k) > 0.5, pick * scale, x).to(dtype)


# ------------------------------------------------------------------------------------------- quantisation
SHAPES = [(1, 1), (1, 32), (3, 7), (5, 33), (31, 64), (32, 31), (33, 100), (64, 128), (65, 129), (127, 255), (130, 2880), (257, 513),
          (2, 4096), (1000, 71), (4, 12345), (129, 8), (300, 1024)]


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", DT)
def test_quantize_shapes(m, k, dtype):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x = rows(m, k, dtype, seed=m * k)
    by_row, by_column = quantized(x), quantized(x.t())
    same(dgm.mxfp4_quantize(x), by_row)
    same(dgm.mxfp4_quantize(x, transpose=True), by_column)
    both = dgm.mxfp4_quantize_both(x)
    same(both[0], by_row)
    same(both[1], by_column)


@pytest.mark.parametrize("dtype", DT)
def test_quantize_strides(dtype):
    """Padded rows, rows off 16 bytes, a transposed view, single columns, a broadcast row."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    big = rows(70, 300, dtype, seed=3)
    for x in (big[:, :256], big[3:, 5:133], big.t(), big[:, 7:8], big[::2, ::3], big[:1].expand(40, 300), big[:, :1].expand(70, 64),
              big.t()[4:100, 8:40]):
        want = quantized(x), quantized(x.t())
        same(dgm.mxfp4_quantize(x), want[0])
        same(dgm.mxfp4_quantize(x, transpose=True), want[1])
        got = dgm.mxfp4_quantize_both(x)
        same(got[0], want[0])
        same(got[1], want[1])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("left", [1, 2, 8])
def test_quantize_rows_of_any_length_between_others(dtype, left):
    """Rows that start and end anywhere, beside NaN that no block may see."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for n in (*range(1, 26), 31, 33, 97, 127, 129, 1021):
        big = torch.full((140, n + left + 9), float("nan"), dtype=dtype, device="cuda")
        x = big[3:136, left:left + n]
        x.copy_(rows(133, n, dtype, seed=n))
        want = quantized(x), quantized(x.t())
        same(dgm.mxfp4_quantize(x), want[0])
        got = dgm.mxfp4_quantize_both(x)
        same(got[0], want[0])
        same(got[1], want[1])
        same(dgm.mxfp4_quantize(x, transpose=True), want[1])


@pytest.mark.parametrize("dtype", DT)
def test_quantize_every_value_beside_a_midpoint(dtype):
    """Midpoints and the numbers next to them in the type, under scales from the type's smallest to its largest."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    bits = {torch.bfloat16: torch.int16, torch.float16: torch.int16, torch.float32: torch.int32}[dtype]
    exps = {torch.bfloat16: range(-120, 125), torch.float16: range(-12, 13), torch.float32: range(-120, 125)}[dtype]
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = torch.stack([(mids.to(dtype).view(bits) + d).view(dtype).double() for d in (-1, 0, 1)]).flatten()      # 21 values
    block = torch.cat([near, -near[:10], torch.tensor([6.0], dtype=torch.float64)])                               # 32
    x = torch.stack([(block * 2.0 ** e).to(dtype) for e in exps]).cuda()
    same(dgm.mxfp4_quantize(x), quantized(x, 0.0) if dtype == torch.float16 else quantized(x))
    same(dgm.mxfp4_quantize(x.t().contiguous(), transpose=True), quantized(x))
    # the largest of a block beside 6 2^e
    six = (torch.tensor([6.0], dtype=dtype).view(bits) + torch.tensor([-1, 0, 1], dtype=bits)).view(dtype)
    x = torch.zeros(3, 32, dtype=dtype)
    x[:, 9] = six
    x = x.cuda()
    got = dgm.mxfp4_quantize(x)
    same(got, quantized(x))
    assert got[1].flatten().tolist() == [127, 127, 128]


def test_quantize_extremes():
    """The largest fp32 numbers, subnormal ones, all zeros, floors, and blocks with infinities and NaN."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x = torch.zeros(8, 96, device="cuda")
    x[0] = torch.finfo(torch.float32).max
    x[1] = -torch.finfo(torch.float32).max / 3
    x[2] = 1e-41
    x[3] = torch.linspace(-1e-30, 1e-30, 96, device="cuda")
    x[4, 40] = float("inf")
    x[4, 41:60] = 3.0
    x[5, 95] = float("nan")
    x[5, :64] = 1.0
    x[6, 3] = -float("inf")
    x[6, 4] = float("nan")
    for floor in (1e-30, 0.0, 1e-4, 6.0, 1e30):
        for t in (x, x.to(torch.bfloat16)):
            same(dgm.mxfp4_quantize(t, amax_floor=floor), quantized(t, floor))
            same(dgm.mxfp4_quantize(t, transpose=True, amax_floor=floor), quantized(t.t(), floor))
    codes, scales = dgm.mxfp4_quantize(x)
    assert scales[4].tolist()[1] == 255 and scales[5].tolist()[2] == 255 and not bool((scales[5, :2] == 255).any())
    assert not bool(codes[4, 16:32].any())


def test_quantize_is_the_layers_cast():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x = rows(70, 512, torch.bfloat16, seed=5)
    for floor in (1e-4, 1e-30):
        packed, sf = dgm.per_token_cast_to_fp4(x, use_packed_ue8m0=True, amax_floor=floor)
        codes, scales = dgm.mxfp4_quantize(x, amax_floor=floor)
        assert torch.equal(packed, codes) and torch.equal(sf.view(torch.uint8), scales)


def test_quantize_empty():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for m, k in ((0, 64), (64, 0), (0, 0)):
        x = torch.zeros((m, k), device="cuda")
        got = dgm.mxfp4_quantize_both(x)
        assert [tuple(t.shape) for p in got for t in p] == [(m, 16 * ((k + 31) // 32)), (m, (k + 31) // 32),
                                                            (k, 16 * ((m + 31) // 32)), (k, (m + 31) // 32)]


def test_quantize_beyond_32_bit_offsets():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x = torch.zeros((40, 1 << 27), dtype=torch.bfloat16, device="cuda")[:, :4096]        # rows 2^28 bytes apart
    x.copy_(rows(40, 4096, torch.bfloat16, seed=9))
    same(dgm.mxfp4_quantize(x), quantized(x))
    same(dgm.mxfp4_quantize(x, transpose=True), quantized(x.t()))


# ------------------------------------------------------------------------------------------- product
def operand(m, k, seed, whole=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (m, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    lo, hi = (127, 129) if whole else (119, 136)
    return codes, torch.randint(lo, hi, (m, k // 32), generator=g, device="cuda", dtype=torch.uint8)


def product(a, b):
    """(value, sum of |products|)"""
    a, b = values(a), values(b).t().contiguous()
    return a @ b, a.abs() @ b.abs()


def check(d, ref, mag, k):
    fi = torch.finfo(d.dtype)
    tol = ref.abs() * (fi.eps / 2) + (145 + k / 128) * 2 * U * mag * (1 + fi.eps) + fi.tiny
    over = ref.abs() + (145 + k / 128) * 2 * U * mag >= fi.max
    bad = ~(((d.double() - ref).abs() <= tol) | (over & torch.isinf(d) & (d.double() * ref > 0)))
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())


def check_swiglu(d, ref, mag, k, clamp):
    (g, u), (gm, um) = ref.chunk(2, 1), mag.chunk(2, 1)
    c = clamp if clamp is not None else float("inf")
    g, u = g.clamp(max=c), u.clamp(-c, c)
    s = torch.sigmoid(g)
    want = g * s * u
    # gate and up off by their sums' share each, the sigmoid's rounding, and results below the least normal number
    off = (145 + k / 128) * 2 * U * (gm * s * (1 + g.abs()) * u.abs() + um * (g * s).abs()) + \
        U * want.abs() * (16 + 8 * g.abs()) + 2.0 ** -126 * (g * u).abs()
    fi = torch.finfo(d.dtype)
    tol = want.abs() * (fi.eps / 2) + 1.01 * off * (1 + fi.eps) + fi.tiny
    over = want.abs() + off >= fi.max
    bad = ~(((d.double() - want).abs() <= tol) | (over & torch.isinf(d)))
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())


GEMMS = [(1, 1, 32), (1, 16, 64), (1, 4096, 2048), (2, 30, 96), (3, 7, 160), (5, 64, 256), (16, 16, 288), (17, 33, 512), (31, 100, 544),
         (33, 257, 1024), (48, 512, 2080), (63, 130, 320), (64, 4096, 7168), (65, 128, 2048), (100, 384, 800), (128, 128, 256),
         (129, 320, 1280), (200, 1000, 192), (255, 513, 544), (256, 256, 512), (300, 2880, 2048), (777, 640, 1312), (1000, 5120, 2880),
         (2049, 1040, 352), (1000, 4000, 1024), (2000, 4002, 1056), (4000, 4000, 1056), (3999, 4034, 800), (64, 64, 65536), (4, 40, 40000)]


@pytest.mark.parametrize("m,n,k", GEMMS)
def test_gemm_exact_sums(m, n, k):
    """Scales of 1 and 2: sums are whole numbers of quarters below 2^24, so nothing may be rounded."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(m, k, m + k, True), operand(n, k, n + k + 1, True)
    ref, mag = product(a, b)
    assert float(mag.max()) * 4 < 2 ** 24 or k > 16384
    d = torch.full((m, n), 7.0, device="cuda")
    assert dgm.mxfp4_gemm_nt(a, b, d) is d
    if float(mag.max()) * 4 < 2 ** 24:
        assert torch.equal(d.double(), ref), torch.nonzero(d.double() != ref)[:4].tolist()
    check(d, ref, mag, k)


@pytest.mark.parametrize("m,n,k", GEMMS)
def test_gemm_shapes(m, n, k):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(m, k, m + k), operand(n, k, n + k + 1)
    torch.manual_seed(m + n)
    ref, mag = product(a, b)
    for dt in DT:
        d = torch.full((m + 1, n + 3), 7.0, dtype=dt, device="cuda")
        dgm.mxfp4_gemm_nt(a, b, d[:m, :n])
        check(d[:m, :n], ref, mag, k)
        assert bool((d[m:] == 7).all()) and bool((d[:, n:] == 7).all())
        d = torch.full((m, n), 7.0, dtype=dt, device="cuda")
        c = (torch.randn((m, n), device="cuda") * 100).to(dt)
        check(dgm.mxfp4_gemm_nt(a, b, d, c=c), ref + c.double(), mag + c.double().abs(), k)
        bias = (torch.randn(n, device="cuda") * 100).to(dt)
        check(dgm.mxfp4_gemm_nt(a, b, d, c=bias), ref + bias.double(), mag + bias.double().abs(), k)
        d.copy_(c)
        check(dgm.mxfp4_gemm_nt(a, b, d, c=d), ref + c.double(), mag + c.double().abs(), k)
    if n % 2 == 0:
        for dt, clamp, fast in ((torch.bfloat16, 10.0, True), (torch.float32, 1.0, False), (torch.float16, 3.0, True)):
            d = torch.full((m, n // 2 + 2), 7.0, dtype=dt, device="cuda")
            dgm.mxfp4_gemm_nt(a, b, d[:, :n // 2], activation="swiglu", activation_clamp=clamp, fast_math=fast)
            check_swiglu(d[:, :n // 2], ref, mag, k, clamp)
            assert bool((d[:, n // 2:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(1, 10, 4096), (1, 34, 8224), (2, 4098, 8256), (3, 2046, 4128), (5, 18, 14016), (7, 1030, 4416),
                                   (8, 2048, 8448), (8, 2050, 4128), (9, 2048, 4096), (2, 8206, 8192), (16, 4090, 2080), (16, 4098, 2080),
                                   (31, 4096, 1056), (50, 1026, 800)])
def test_gemm_few_tokens(m, n, k):
    """The forms that few tokens take: parts of K in a fragment, gate and up rows in one or two, edges in every direction."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for whole in (True, False):
        a, b = operand(m, k, m + k, whole), operand(n, k, n + k + 1, whole)
        ref, mag = product(a, b)
        f = torch.full((m + 1, n + 3), 7.0, device="cuda")
        dgm.mxfp4_gemm_nt(a, b, f[:m, :n])
        check(f[:m, :n], ref, mag, k)
        if whole:
            assert torch.equal(f[:m, :n].double(), ref)
        assert bool((f[:, n:] == 7).all()) and bool((f[m:] == 7).all())
        d = torch.full((m + 1, n // 2), 7.0, dtype=torch.bfloat16, device="cuda")
        check_swiglu(dgm.mxfp4_gemm_nt(a, b, d[:m], activation="swiglu", activation_clamp=3.0), ref, mag, k, 3.0)
        assert bool((d[m:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(69, 8278, 288), (200, 8242, 320), (392, 8206, 288), (586, 8292, 288), (4100, 1830, 288),
                                   (1025, 7226, 288), (1732, 6474, 288), (50, 4246, 8224), (18, 7758, 8224), (65, 8270, 14368),
                                   (67, 4354, 14368), (133, 5502, 14368), (135, 8284, 20512), (225, 8230, 20512), (585, 4106, 32800)])
def test_gemm_ragged_tiles(m, n, k):
    """The tile sizes that wide outputs and long sums take, whole and in ranges of K, with edges in every direction."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(m, k, m + k), operand(n, k, n + k + 1)
    ref, mag = product(a, b)
    d = torch.full((m + 1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    bias = torch.randn(n, device="cuda").to(torch.bfloat16)
    check(dgm.mxfp4_gemm_nt(a, b, d[:m], c=bias), ref + bias.double(), mag + bias.double().abs(), k)
    assert bool((d[m:] == 7).all())
    first = d.clone()
    assert torch.equal(dgm.mxfp4_gemm_nt(a, b, d[:m], c=bias), first[:m])            # (the same bits again)
    d = torch.full((m + 1, n // 2), 7.0, dtype=torch.bfloat16, device="cuda")
    check_swiglu(dgm.mxfp4_gemm_nt(a, b, d[:m], activation="swiglu", activation_clamp=2.0), ref, mag, k, 2.0)
    assert bool((d[m:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (20, 48, 96), (40, 96, 544), (130, 200, 544), (300, 512, 2080), (600, 4096, 1024)])
def test_gemm_nan_scales(m, n, k):
    """A block of scale 255 makes the results of its row NaN and no others."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(m, k, 1), operand(n, k, 2)
    bad_m, bad_n = m // 2, n // 3
    a[1][bad_m, k // 32 - 1] = 255
    a[0][bad_m] = 0                        # (as the quantiser leaves them: zeros)
    b[1][bad_n, 0] = 255
    ref, mag = product(a, b)
    d = dgm.mxfp4_gemm_nt(a, b, torch.zeros((m, n), device="cuda"))
    want = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    want[bad_m] = True
    want[:, bad_n] = True
    assert torch.equal(torch.isnan(d), want)
    check(torch.where(want, torch.zeros_like(d), d), torch.where(want, 0, ref), torch.where(want, 0, mag), k)
    d = dgm.mxfp4_gemm_nt(a, b, torch.zeros((m, n // 2), device="cuda"), activation="swiglu", activation_clamp=None)
    assert bool(torch.isnan(d[bad_m]).all()) and bool(torch.isnan(d[:, bad_n % (n // 2)]).all())


@pytest.mark.parametrize("m", [1, 7, 30, 100, 700])
def test_gemm_operands_as_they_come(m):
    """Code rows off 16 bytes, in padded memory and as views, scales in rows of any stride and as int32 words, c in other
    strides, repeated rows, a quantiser's own rows."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    n, k = 80, 384
    a, b = operand(m, k, 11), operand(n, k, 12)
    ref, mag = product(a, b)
    run = lambda a, b, **kw: dgm.mxfp4_gemm_nt(a, b, torch.zeros((m, n), device="cuda"), **kw)
    plain = run(a, b)
    check(plain, ref, mag, k)

    def padded(t, left, right):
        big = torch.full((t.size(0), t.size(1) + left + right), 99, dtype=torch.uint8, device="cuda")
        big[:, left:left + t.size(1)] = t
        return big[:, left:left + t.size(1)]
    for left, right in ((16, 16), (1, 0), (0, 5), (3, 13)):
        assert torch.equal(run((padded(a[0], left, right), padded(a[1], left, right)), (padded(b[0], right, left), padded(b[1], right, left))), plain)
    column = lambda t: t.t().contiguous().t()
    assert torch.equal(run((column(a[0]), column(a[1])), (column(b[0]), column(b[1]))), plain)
    assert torch.equal(run((a[0], a[1].view(torch.int32)), (b[0], b[1].view(torch.int32))), plain)
    c = torch.randn((n, m), device="cuda").t()
    assert torch.equal(run(a, b, c=c), run(a, b, c=c.contiguous()))
    one = a[0][:1].expand(m, k // 2), a[1][:1].expand(m, k // 32)
    assert torch.equal(run(one, b), plain[:1].expand(m, n))
    x = torch.randn((m, 400), device="cuda").to(torch.bfloat16)
    w = torch.randn((n, 400), device="cuda").to(torch.bfloat16)
    qa, qb = dgm.mxfp4_quantize(x), dgm.mxfp4_quantize(w)
    ref, mag = product(quantized(x), quantized(w))
    check(run(qa, qb), ref, mag, 416)


def test_gemm_beyond_32_bit_offsets():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for m in (20, 200):
        a, b = operand(m, 512, 21), operand(300, 512, 22)
        wide = torch.zeros((300, 1 << 24), dtype=torch.uint8, device="cuda")[:, :256]
        wide.copy_(b[0])
        d = torch.zeros((m, (1 << 31) // m + 64), dtype=torch.bfloat16, device="cuda")[:, :300]
        ref, mag = product(a, b)
        check(dgm.mxfp4_gemm_nt(a, (wide, b[1]), d), ref, mag, 512)


def test_gemm_on_another_stream_and_in_a_graph():
    """Two products with a workspace each, on two streams at once and replayed."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(64, 8192, 31), operand(1024, 8192, 32)
    a2 = operand(100, 8192, 33)
    want, want2 = (dgm.mxfp4_gemm_nt(x, b, torch.zeros((x[0].size(0), 1024), device="cuda")).clone() for x in (a, a2))
    d, d2 = torch.zeros_like(want), torch.zeros_like(want2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(s):
            dgm.mxfp4_gemm_nt(a2, b, d2)
        dgm.mxfp4_gemm_nt(a, b, d)
    torch.cuda.synchronize()
    assert torch.equal(d, want) and torch.equal(d2, want2)
    graph = torch.cuda.CUDAGraph()
    x, w = torch.randn((64, 8192), device="cuda"), torch.randn((1024, 8192), device="cuda")

    def run():
        q, qt = dgm.mxfp4_quantize_both(x)
        y = dgm.mxfp4_gemm_nt(q, dgm.mxfp4_quantize(w), d)
        return y, qt[0], dgm.mxfp4_linear_backward(y, qt, dgm.mxfp4_quantize(w, transpose=True), x.shape, w.shape)
    run()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        x.normal_()
        w.normal_()
        graph.replay()
        torch.cuda.synchronize()
        y, qt, grads = (held[0].clone(), held[1].clone(), [t.clone() for t in held[2]])
        eager = run()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[0]) and torch.equal(qt, eager[1]) and all(torch.equal(p, q) for p, q in zip(grads, eager[2])), i


# ------------------------------------------------------------------------------------------- linear
def q64(x):
    return values(quantized(x))


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 96), (5, 33, 70), (64, 128, 256), (100, 40, 31), (257, 300, 513), (777, 1234, 640)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float32, torch.bfloat16)])
def test_linear(m, n, k, dtype, wdtype):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    torch.manual_seed(m + n + k)
    x = torch.randn((m, k), device="cuda").to(dtype).requires_grad_()
    w = (torch.randn((n, k), device="cuda") * 0.1).to(wdtype).requires_grad_()
    dy = (torch.randn((m, n), device="cuda") * 1e-3).to(dtype)
    y = dgm.mxfp4_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == wdtype
    pad = lambda v: (v + 31) // 32 * 32
    for got, a, b, inner in ((y, x, w, k), (dx, dy, w.t(), n), (dw, dy.t(), x.t(), m)):
        a, b = q64(a.detach()), q64(b.detach()).t().contiguous()
        check(got.detach(), a @ b, a.abs() @ b.abs(), pad(inner))
    # the explicit calls, one gradient at a time, and without autograd
    y2, xt, wt = dgm.mxfp4_linear_forward(x, w)
    assert not y2.requires_grad and torch.equal(y2, y)
    got = dgm.mxfp4_linear_backward(dy, xt, wt, x.shape, w.shape, w.dtype)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    for needs in ((True, False), (False, True)):
        y2, xt, wt = dgm.mxfp4_linear_forward(x, w, needs=needs)
        assert (xt is None) == (not needs[1]) and (wt is None) == (not needs[0])
        got = dgm.mxfp4_linear_backward(dy, xt, wt, x.shape, w.shape, w.dtype, needs=needs)
        assert (got[0] is None or torch.equal(got[0], dx)) and (got[1] is None or torch.equal(got[1], dw))
    with torch.no_grad():
        assert torch.equal(dgm.mxfp4_linear(x, w), y)
    for leaf in (x, w):
        xs, ws = x.detach(), w.detach()
        (xs if leaf is x else ws).requires_grad_()
        g = torch.autograd.grad(dgm.mxfp4_linear(xs, ws), xs if leaf is x else ws, dy)[0]
        assert torch.equal(g, dx if leaf is x else dw)


def test_linear_where_nothing_is_rounded():
    """Operands that MXFP4 holds along both dimensions: the gradients are those of the product, and its differences
    (a product's are linear: steps of any size)."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    g = torch.Generator(device="cuda").manual_seed(3)
    lv = torch.tensor(LEVELS, device="cuda")

    def exact(m, k):
        t = lv[torch.randint(0, 8, (m, k), generator=g, device="cuda")] * torch.where(torch.rand((m, k), generator=g, device="cuda") > 0.5, 1.0, -1.0)
        i = torch.arange(min(m, k), device="cuda")
        for s in range(0, max(m, k), 32):          # (a six in every block of 32, either way)
            t[i % m, (i + s) % k] = 6.0
            t[(i + s) % m, i % k] = 6.0
        return t
    x, w, dy = exact(64, 96), exact(128, 96), exact(64, 128)
    assert all(torch.equal(q64(t), t.double()) and torch.equal(q64(t.t()), t.t().double()) for t in (x, w, dy))
    x.requires_grad_()
    w.requires_grad_()
    y = dgm.mxfp4_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xd, wd, dyd = x.detach().double(), w.detach().double(), dy.double()
    assert torch.equal(y.detach().double(), xd @ wd.t().contiguous())
    assert torch.equal(dx.double(), dyd @ wd) and torch.equal(dw.double(), dyd.t().contiguous() @ xd)
    f = lambda x, w: float((dgm.mxfp4_linear(x, w).double() * dyd).sum())
    with torch.no_grad():
        base = f(x, w)
        for i, j in ((0, 1), (17, 40), (63, 95)):
            step = x.clone()
            step[i, j] = 0.0 if float(x[i, j]) else 1.0
            if torch.equal(q64(step), step.double()):
                assert f(step, w) - base == float(dx[i, j]) * float(step[i, j] - x[i, j])


def test_linear_shared_and_broadcast_leaves():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    torch.manual_seed(4)
    w = (torch.randn((64, 64), device="cuda") * 0.1).requires_grad_()
    x = torch.randn((32, 64), device="cuda")
    h = dgm.mxfp4_linear(x, w)
    y = dgm.mxfp4_linear(h, w)                                   # the same weight twice
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, w, dy)[0]
    hd = h.detach()
    dh, dw2 = dgm.mxfp4_linear_backward(dy, *dgm.mxfp4_linear_forward(hd, w.detach())[1:], hd.shape, w.shape)
    _, dw1 = dgm.mxfp4_linear_backward(dh, *dgm.mxfp4_linear_forward(x, w.detach())[1:], x.shape, w.shape)
    assert torch.equal(got, dw1 + dw2) or torch.equal(got, dw2 + dw1)
    row = torch.randn((1, 64), device="cuda", requires_grad=True)        # one row for all tokens
    y = dgm.mxfp4_linear(row.expand(40, 64), w)
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, row, dy)[0]
    full = dgm.mxfp4_linear_backward(dy, None, dgm.mxfp4_quantize(w.detach(), transpose=True), (40, 64), w.shape, needs=(True, False))[0]
    assert torch.allclose(got, full.sum(0, keepdim=True), rtol=0, atol=float(full.abs().sum(0).max()) * 40 * U)


def test_linear_no_tokens_and_refusals():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x = torch.zeros((0, 64), device="cuda", requires_grad=True)
    w = torch.ones((32, 64), device="cuda", requires_grad=True)
    y = dgm.mxfp4_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 32) and dx.shape == (0, 64) and not bool(dw.any())
    x = torch.ones((4, 64), device="cuda", requires_grad=True)
    y = dgm.mxfp4_linear(x, w)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="under graph capture"):
        with torch.cuda.graph(graph):
            dgm.mxfp4_linear(x, w)


def test_quantize_more_workgroups_than_one_axis():
    """2^23 and more workgroups: one row repeated, so that its codes are known."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x = rows(1, 2048, torch.bfloat16, seed=4)
    want = quantized(x)
    n = (1 << 23) + 3
    codes, scales = dgm.mxfp4_quantize(x.expand(n, 2048))
    for part in (codes[:2], codes[-5:], codes[(1 << 23) - 2:]):
        assert bool((part == want[0]).all())
    assert bool((codes.view(torch.int64) == want[0].view(torch.int64)).all()) and bool((scales == want[1]).all())
