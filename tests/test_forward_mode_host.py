"""Forward-mode tangents (CPU, launches left out): refused, not dropped."""
import types

import pytest
import torch
from torch.autograd import forward_ad

import hopper_megamoe_basedondeepgemm_amd as dgm
from tests.no_launch import no_launch  # noqa: F401


def norm_args():
    return dict(x=torch.randn(4, 16), residual=torch.randn(4, 16), post_weight=torch.ones(16), pre_weight=torch.ones(16),
                gate=torch.ones(4, 1))


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("name", ["x", "residual", "post_weight", "pre_weight", "gate"])
def test_norm(no_launch, name):  # noqa: F811
    a = norm_args()
    dgm.rms_norm_residual(**a)
    with forward_ad.dual_level():
        dgm.rms_norm_residual(**a)                            # (a level alone is nothing to refuse)
        a[name] = dual(a[name])
        for call in (dgm.rms_norm_residual, dgm.rms_norm_residual_forward):
            with pytest.raises(RuntimeError, match="tangent"):
                call(**a)
        with pytest.raises(RuntimeError, match="tangent"):
            dgm.rms_norm_residual_backward(torch.ones(4, 16), None, a["x"], a["residual"], torch.ones(4), torch.ones(4),
                                           a["post_weight"], a["pre_weight"], a["gate"])
    assert len(no_launch.calls) == 2


def test_norm_outputs_and_gradients(no_launch):  # noqa: F811
    a = norm_args()
    with forward_ad.dual_level():
        for name in ("residual_out", "out"):
            with pytest.raises(RuntimeError, match="tangent"):
                dgm.rms_norm_residual(**a, **{name: dual(torch.zeros(4, 16))})
        with pytest.raises(RuntimeError, match="tangent"):
            dgm.rms_norm_residual_backward(dual(torch.ones(4, 16)), None, a["x"], a["residual"], torch.ones(4), torch.ones(4),
                                           a["post_weight"], a["pre_weight"], a["gate"])
        leaf = a["x"].requires_grad_()
        r, h = dgm.rms_norm_residual(**a)
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad((r, h), leaf, (dual(torch.ones(4, 16)), torch.ones(4, 16)))


def test_balance(no_launch):  # noqa: F811
    logits, idx = torch.randn(5, 8), torch.zeros((5, 2), dtype=torch.int64)
    _, counts, stats = dgm.router_balance_loss_forward(logits, idx)
    with forward_ad.dual_level():
        for call in (dgm.router_balance_loss, dgm.router_balance_loss_forward):
            with pytest.raises(RuntimeError, match="tangent"):
                call(dual(logits), idx)
        with pytest.raises(RuntimeError, match="tangent"):
            dgm.router_balance_loss_backward(dual(torch.ones(())), logits, idx, counts, stats)
        loss, _ = dgm.router_balance_loss(logits.requires_grad_(), idx)
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(loss, logits, dual(torch.ones(())))


@pytest.mark.parametrize("name", ["sfa", "sfb", "c", "d"])
def test_int8_gemm(no_launch, name):  # noqa: F811
    t = dict(sfa=torch.ones(4), sfb=torch.ones(8), c=torch.zeros(4, 8), d=torch.zeros(4, 8))
    a, b = torch.zeros((4, 32), dtype=torch.int8), torch.zeros((8, 32), dtype=torch.int8)
    with forward_ad.dual_level():
        t[name] = dual(t[name])
        with pytest.raises(RuntimeError, match="tangent"):
            dgm.int8_gemm_nt((a, t["sfa"]), (b, t["sfb"]), t["d"], c=t["c"])
    assert not no_launch.calls


def test_block(no_launch):  # noqa: F811
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    buffer = types.SimpleNamespace(hidden=32, num_experts=4, num_local_experts=4)
    with forward_ad.dual_level():
        for kw in (dict(gate=dual(bf(4, 1))), dict(next_weight=dual(bf(32))), dict(post_weight=dual(bf(32)))):
            with pytest.raises(RuntimeError, match="tangent"):
                dgm.mega_moe_block(bf(4, 32), bf(32), bf(4, 32), None, None, buffer, **kw)
    assert not no_launch.calls
