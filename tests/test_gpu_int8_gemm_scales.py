"""int8_gemm_nt with scales that are no numbers or infinite."""
import pytest
import torch

from tests.gpu_common import need_gpu
from tests.test_gpu_int8_gemm import make, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (2, 96, 4352), (16, 128, 512), (40, 96, 528), (33, 50, 37), (64, 4096, 7168), (300, 320, 1024)])
def test_infinite_and_nan_scales(m, n, k):
    """They reach the result: NaN where the formula has it, in SwiGLU's clamped halves too."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    a, b = make(m, n, k, seed=m + n + k)
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")
    a[1][:3] = bad[:min(m, 3)]
    b[1][1:4], b[1][n // 2 + 2:n // 2 + 5] = bad, bad
    ref = product(a, b)
    for clamp in (10.0, None):
        d = torch.zeros((m, n // 2), device="cuda")
        dgm.int8_gemm_nt(a, b, d, activation="swiglu", activation_clamp=clamp)
        g, u = ref.chunk(2, 1)
        if clamp is not None:
            g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
        want = g * torch.sigmoid(g) * u
        assert torch.equal(torch.isnan(d), torch.isnan(want)) and bool(torch.isnan(want).any())
        over = want.abs() > torch.finfo(torch.float32).max
        assert torch.equal(d.double()[over].sign(), want[over].sign()) and bool(torch.isinf(d[over]).all())
        assert bool(torch.isfinite(d[~over & ~torch.isnan(want)]).all())
    d = torch.zeros((m, n), device="cuda")
    dgm.int8_gemm_nt(a, b, d)
    assert torch.equal(torch.isnan(d), torch.isnan(ref)) and torch.equal(torch.isinf(d), torch.isinf(ref))
