"""Saved tensors that hooks bring back as something else (CPU, launches left out): the backward pass reads their
memory by address, so it refuses other types and shapes before it does."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm
from tests.no_launch import no_launch  # noqa: F401


def hooks(change):
    """Everything comes back in other memory; what `change` picks, changed."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t.clone()))


def norm(change, **kw):
    x = torch.randn(6, 16, requires_grad=True)
    args = dict(residual=torch.randn(6, 16, requires_grad=True), post_weight=torch.ones(16), pre_weight=torch.ones(16),
                gate=torch.ones(16))
    with hooks(change):
        r, h = dgm.rms_norm_residual(x, **{**args, **kw})
    torch.autograd.grad((r, h), x, (torch.ones_like(r), torch.ones_like(h)))


@pytest.mark.parametrize("change", [
    lambda t: t.bfloat16() if t.shape == (6, 16) else t,           # the rows, at half the bytes
    lambda t: t[:3] if t.shape == (6, 16) else t,                  # half the rows
    lambda t: t[:, :8] if t.shape == (6, 16) else t,
    lambda t: t[:8] if t.shape == (16,) else t,                    # weights and gate
    lambda t: t.half() if t.shape == (16,) else t,
    lambda t: t.half() if t.shape == (2, 6) else t,                # the rstd rows
    lambda t: t[:1] if t.shape == (2, 6) else t,
    lambda t: t[:, :3] if t.shape == (2, 6) else t,
])
def test_norm(no_launch, change):  # noqa: F811
    norm(lambda t: t)
    assert no_launch.calls == ["dgm_rms_norm_residual", "dgm_rms_norm_residual_backward"]
    no_launch.calls.clear()
    with pytest.raises((TypeError, ValueError)):
        norm(change)
    assert no_launch.calls == ["dgm_rms_norm_residual"]


def balance(change):
    logits = torch.randn(300, 8, requires_grad=True)
    with hooks(change):
        loss, _ = dgm.router_balance_loss(logits, torch.zeros((300, 2), dtype=torch.int64),
                                          torch.tensor([0, 100, 200, 300], dtype=torch.int32))
    return torch.autograd.grad(loss, logits)[0]


@pytest.mark.parametrize("change", [
    lambda t: t.bfloat16() if t.shape == (300, 8) else t,          # logits, at half the bytes
    lambda t: t[:, :4] if t.shape == (300, 8) else t,
    lambda t: t[:200] if t.shape == (300, 8) else t,
    lambda t: t.short() if t.shape == (300, 2) else t,             # topk_idx
    lambda t: t[:200] if t.shape == (300, 2) else t,
    lambda t: t.short() if t.shape == (4,) else t,                 # cu_seqlens
    lambda t: t[:3] if t.shape == (4,) else t,
    lambda t: t.short() if t.shape == (3, 8) else t,               # counts
    lambda t: t[:2] if t.shape == (3, 8) else t,
    lambda t: t.short() if t.shape == (16,) else t,                # stats
    lambda t: t[:12] if t.shape == (16,) else t,
])
def test_balance(no_launch, change):  # noqa: F811
    assert balance(lambda t: t).shape == (300, 8)
    assert no_launch.calls == ["dgm_router_balance_loss", "dgm_router_balance_loss_backward"]
    no_launch.calls.clear()
    with pytest.raises((TypeError, ValueError)):
        balance(change)
    assert no_launch.calls == ["dgm_router_balance_loss"]
