"""mega_moe_block with an MXFP4 dense expert and layer norms: what is refused before any GPU work (CPU)."""
import types

import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def rows(m, k):
    return torch.zeros((m, k // 2), dtype=torch.uint8), torch.zeros((m, k // 32), dtype=torch.uint8)


def block(**kw):
    buffer = types.SimpleNamespace(hidden=64, num_experts=4, num_local_experts=4, ep_size=1)
    return dgm.mega_moe_block(bf(4, 64), bf(64), bf(4, 64), None, None, buffer, **kw)


int8 = lambda m, k: (torch.zeros((m, k), dtype=torch.int8), torch.zeros(m))


@pytest.mark.parametrize("kw, err, what", [
    (dict(shared_expert=(rows(64, 64), rows(64, 96))), ValueError, "shared_expert"),
    (dict(shared_expert=(rows(192, 96), rows(64, 96))), ValueError, "shared_expert"),
    (dict(shared_expert=(rows(192, 64), rows(32, 96))), ValueError, "shared_expert"),
    (dict(shared_expert=(rows(0, 64), rows(64, 0))), ValueError, "shared_expert"),
    (dict(shared_expert=((rows(192, 64)[0], rows(191, 64)[1]), rows(64, 96))), TypeError, "gate and up: uint8 scales"),
    (dict(shared_expert=(rows(192, 64), (rows(64, 96)[0], torch.zeros(64)))), TypeError, "down: uint8 scales"),
    (dict(shared_expert=(rows(256, 64), int8(64, 128))), TypeError, "int8"),
    (dict(shared_expert=(int8(256, 64), rows(64, 128))), TypeError, "int8"),
    (dict(shared_expert=(rows(192, 64), rows(64, 96)), activation_clamp=-1.0), ValueError, "activation_clamp"),
    (dict(shared_expert=(rows(192, 64), rows(64, 96))), RuntimeError, "GPU"),
    (dict(norm="batch"), ValueError, "norm 'batch'"),
    (dict(norm_bias=bf(64)), ValueError, "norm='layer'"),
    (dict(next_bias=bf(64)), ValueError, "norm='layer'"),
    (dict(norm="layer", post_weight=bf(64)), ValueError, "no post_weight"),
    (dict(norm="layer", gate=bf(64)), ValueError, "no post_weight and no gate"),
    (dict(norm="layer", next_bias=bf(64)), ValueError, "without a next_weight"),
    (dict(norm="layer", norm_bias=bf(63)), TypeError, "weight and bias"),
    (dict(norm="layer", norm_bias=torch.zeros(64)), TypeError, "weight and bias"),
    (dict(norm="layer", next_weight=bf(64), next_bias=torch.zeros(64)), TypeError, "weight and bias"),
    (dict(norm="layer", residual=bf(4, 65)), TypeError, "rows of"),
    (dict(norm="layer", norm_bias=bf(64).requires_grad_()), RuntimeError, "no gradient"),
    (dict(norm="layer", norm_bias=bf(64), next_weight=bf(64), next_bias=bf(64)), RuntimeError, "GPU"),
])
def test_refusals_come_before_the_layer(kw, err, what, monkeypatch):
    from hopper_megamoe_basedondeepgemm_amd import block as module
    monkeypatch.setattr(module, "mxfp4_mega_moe_from_bf16", lambda *a, **k: pytest.fail("the layer has run"))
    for name in ("_norm", "_layer_norm"):
        monkeypatch.setattr(module, name, lambda *a, **k: pytest.fail("a norm has run"))
    with pytest.raises(err, match=what):
        block(**kw)
