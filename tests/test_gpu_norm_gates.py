"""Sigmoid gates of rms_norm_residual far from zero: their complement and their small values."""
import pytest
import torch

from tests.gpu_common import need_gpu
from tests.test_gpu_norm import Form, U, close, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate", ["channel", "token", "full"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H", [96, 100, 2880, 16384])
def test_gradient_of_a_wide_open_gate(gate, dtype, H):
    """sigmoid'(g) = sigmoid(g) sigmoid(-g), relative to itself where sigmoid(g) rounds to 1: each factor within
    (6 + |g|) 2^-24 (|g| up to 30: 72 for both), beside the 256 of a gradient and the terms of its sum."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    T = 40
    x, r, w1, w2, gt = make(T, H, dtype, torch.float32, 1, 1, gate, 1, seed=H)
    gt = torch.linspace(-30, 30, gt.numel(), device="cuda").to(dtype).view(gt.shape).requires_grad_()
    got_r, got_h = dgm.rms_norm_residual(x, r, w1, w2, gt, True, 0.5)
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    (got,) = torch.autograd.grad((got_r, got_h), gt, (dr, dh))
    f = Form(x, r, w1, w2, gt, True, 0.5)
    # R' and its magnitude from the residual's gradient; then s R' n sigmoid(g) sigmoid(-g)
    R, Rm = f.grads(dr, dh)["residual"]
    g = gt.detach().double()
    k = (torch.sigmoid(g) * torch.sigmoid(-g)).expand_as(R)
    value, mag = f.over(0.5 * R * f.n * k), f.over(0.5 * Rm * f.n.abs() * k)
    over = T if value.dim() == 1 else H if value.shape != R.shape else 0
    # (below the least normal number a type has a fixed step)
    fi = torch.finfo(dtype)
    off = (got.double() - value).abs()
    tol = value.abs() * (fi.eps / 2) + (256 + 72 + over) * U * mag * (1 + fi.eps) + fi.tiny * fi.eps
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("gate", ["channel", "token", "full"])
def test_small_gates_of_fp32_rows(gate):
    """fp32 rows: sigmoid within 8 2^-24 of itself wherever it is a normal number (the hardware's exponential and
    reciprocal within a unit, 2 2^-24, each; the exponential's correction, the sum and the product half a unit each; 1
    for the exponent's last bits)."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    T, H = 64, 64
    x = torch.ones((T, H), device="cuda")
    shape = {"channel": (H,), "token": (T, 1), "full": (T, H)}[gate]
    n = T * H if gate == "full" else 64
    for lo, hi in ((-86, -40), (-40, 0), (0, 90)):
        g = torch.linspace(lo, hi, n, device="cuda").view(shape)
        r, _ = dgm.rms_norm_residual(x, gate=g, gate_sigmoid=True)
        want = torch.sigmoid(g.double()).expand(T, H)
        assert bool(((r.double() - want).abs() <= 8 * U * want).all()), float(((r.double() - want).abs() / want).max() / U)
