"""mxfp4_gemm_nt against its definition in 64 bits, through every kernel that the host chooses from (tests/mxfp4_forms.py)
and with results of many tiles a CU. Tolerances as derived in tests/test_gpu_mxfp4.py."""
import pytest
import torch

from tests.gpu_common import need_gpu
from tests.mxfp4_forms import PLAIN, SWIGLU
from tests.test_gpu_mxfp4 import check, check_swiglu, operand, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [s for some in PLAIN.values() for s in some])
def test_every_form(m, n, k):
    """Whole sums without a rounding; then any scales with nothing added, a bias and d itself, in rows between others."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(m, k, m + k, True), operand(n, k, n + k + 1, True)
    ref, mag = product(a, b)
    d = torch.full((m + 1, n + 3), 7.0, device="cuda")
    dgm.mxfp4_gemm_nt(a, b, d[:m, :n])
    check(d[:m, :n], ref, mag, k)
    if float(mag.max()) * 4 < 2 ** 24:
        assert torch.equal(d[:m, :n].double(), ref), torch.nonzero(d[:m, :n].double() != ref)[:4].tolist()
    assert bool((d[m:] == 7).all()) and bool((d[:, n:] == 7).all())
    a, b = operand(m, k, m + k), operand(n, k, n + k + 1)
    ref, mag = product(a, b)
    g = torch.Generator(device="cuda").manual_seed(m + n)
    d = torch.full((m + 1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    bias = (torch.randn(n, generator=g, device="cuda") * 100).to(torch.bfloat16)
    check(dgm.mxfp4_gemm_nt(a, b, d[:m], c=bias), ref + bias.double(), mag + bias.double().abs(), k)
    first = d.clone()
    assert torch.equal(dgm.mxfp4_gemm_nt(a, b, d[:m], c=bias), first[:m]) and bool((d[m:] == 7).all())
    c = (torch.randn((m, n), generator=g, device="cuda") * 100).to(torch.float16)
    d = c.clone()
    check(dgm.mxfp4_gemm_nt(a, b, d, c=d), ref + c.double(), mag + c.double().abs(), k)


@pytest.mark.parametrize("m,n,k", [s for some in SWIGLU.values() for s in some])
def test_every_form_with_swiglu(m, n, k):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(m, k, m + k), operand(n, k, n + k + 1)
    ref, mag = product(a, b)
    for dt, clamp, fast in ((torch.bfloat16, 10.0, True), (torch.float32, 1.0, False), (torch.float16, 3.0, True)):
        d = torch.full((m + 1, n // 2 + 3), 7.0, dtype=dt, device="cuda")
        check_swiglu(dgm.mxfp4_gemm_nt(a, b, d[:m, :n // 2], activation="swiglu", activation_clamp=clamp, fast_math=fast), ref, mag, k, clamp)
        assert bool((d[m:] == 7).all()) and bool((d[:, n // 2:] == 7).all())
        first = d.clone()
        dgm.mxfp4_gemm_nt(a, b, d[:m, :n // 2], activation="swiglu", activation_clamp=clamp, fast_math=fast)
        assert torch.equal(d, first)


@pytest.mark.parametrize("m,n,k,dtype,right", [
    (5003, 5001, 288, torch.float32, 0), (5003, 5001, 288, torch.float32, 3), (7171, 7173, 96, torch.bfloat16, 1),
    (7171, 7173, 96, torch.float16, 0), (390001, 129, 64, torch.bfloat16, 1), (257, 200003, 64, torch.bfloat16, 5)])
def test_results_of_100_megabytes(m, n, k, dtype, right):
    """Rows on 4 bytes and off them: whole pieces, edges in both directions, C added, over d itself."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    assert m * n * torch.empty(0, dtype=dtype).element_size() >= 100000000
    a, b = operand(m, k, 1), operand(n, k, 2)
    ref, mag = product(a, b)
    d = torch.full((m + 1, n + right), 7.0, dtype=dtype, device="cuda")
    check(dgm.mxfp4_gemm_nt(a, b, d[:m, :n]), ref, mag, k)
    g = torch.Generator(device="cuda").manual_seed(3)
    d[:m, :n].normal_(generator=g)
    c = d[:m, :n].double()
    check(dgm.mxfp4_gemm_nt(a, b, d[:m, :n], c=d[:m, :n]), ref + c, mag + c.abs(), k)
    assert bool((d[m:] == 7).all()) and bool((d[:, n:] == 7).all())


def test_results_of_100_megabytes_with_swiglu():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    m, n, k = 7171, 14348, 96
    a, b = operand(m, k, 1), operand(n, k, 2)
    ref, mag = product(a, b)
    d = torch.full((m + 1, n // 2 + 2), 7.0, dtype=torch.bfloat16, device="cuda")
    check_swiglu(dgm.mxfp4_gemm_nt(a, b, d[:m, :n // 2], activation="swiglu", activation_clamp=3.0), ref, mag, k, 3.0)
    assert bool((d[m:] == 7).all()) and bool((d[:, n // 2:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (9, 130, 4128), (40, 96, 544), (130, 200, 544), (66, 129, 5152), (700, 4096, 1024)])
def test_scales_of_every_size(m, n, k):
    """Bytes from 0 to 254 whose product is an ordinary number, or below the least normal one: no rounding but the sum's."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = operand(m, k, 1, True), operand(n, k, 2, True)
    ones = (a[0], torch.full_like(a[1], 127)), (b[0], torch.full_like(b[1], 127))
    ref, mag = product(*ones)
    assert float(mag.max()) * 4 < 2 ** 24
    for sa in (0, 1, 20, 100, 127, 200, 253, 254):
        for total in (120, 254, 330):
            if not 0 <= total - sa <= 254:
                continue
            a[1].fill_(sa)
            b[1].fill_(total - sa)
            d = dgm.mxfp4_gemm_nt(a, b, torch.full((m, n), 7.0, device="cuda"))
            assert torch.equal(d.double(), ref * 2.0 ** (total - 254)), (sa, total)
