"""mega_moe_block: what is refused before any GPU work (CPU)."""
import types

import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def buffer(ep_size=1, hidden=32, experts=4):
    return types.SimpleNamespace(hidden=hidden, num_experts=experts, num_local_experts=experts // ep_size, ep_size=ep_size)


def block(sym_buffer=None, **kw):
    return dgm.mega_moe_block(bf(4, 32), kw.pop("norm_weight", bf(32)), bf(4, 32), None, None, sym_buffer or buffer(), **kw)


def test_an_expert_parallel_share_is_refused():
    """y holds this rank's experts alone there: the norm behind it, the dense expert and the residual belong behind the
    sum over ranks."""
    with pytest.raises(ValueError, match="expert"):
        block(buffer(ep_size=2))
    with pytest.raises(RuntimeError, match="GPU"):
        block()


@pytest.mark.parametrize("name", ["post_wieght", "gate_sigmod", "residul", "num_tokens"])
def test_unknown_options_are_refused(name):
    """The layer's entry point drops names that it does not know; a misspelt part of the block must not vanish there."""
    with pytest.raises(TypeError, match=name):
        block(**{name: None})


def test_an_option_that_nothing_honours_is_refused():
    with pytest.raises(ValueError, match="fast_math"):
        block(fast_math=False)
    with pytest.raises(RuntimeError, match="GPU"):
        block(fast_math=True)


def test_the_layer_gets_its_options(monkeypatch):
    from hopper_megamoe_basedondeepgemm_amd import block as module
    seen = {}

    def layer(y, hidden_states, router_weight, l1, l2, b, cumulative_local_expert_recv_stats=None, activation_clamp=10.0,
              force_balanced=None, token_offset=0, phase_stamps=None, one_launch=None, **_):
        seen.update(stats=cumulative_local_expert_recv_stats, clamp=activation_clamp, balanced=force_balanced,
                    offset=token_offset, stamps=phase_stamps, one=one_launch)
    monkeypatch.setattr(module, "mxfp4_mega_moe_from_bf16", layer)
    monkeypatch.setattr(module, "_norm", lambda x, *a: (x, x, None, None, None, None, None))
    monkeypatch.setattr("hopper_megamoe_basedondeepgemm_amd._lib.require_one_device", lambda *tensors: None)
    block(cumulative_local_expert_recv_stats=1, activation_clamp=2.0, force_balanced=True, token_offset=3, phase_stamps=4,
          one_launch=False)
    assert seen == dict(stats=1, clamp=2.0, balanced=True, offset=3, stamps=4, one=False)


def expert(inner=128, hidden=32, up=None, out=None, dtype=torch.int8):
    up, out = up or 2 * inner, out or 32
    return ((torch.zeros((up, hidden), dtype=dtype), torch.zeros(up)), (torch.zeros((out, inner), dtype=torch.int8), torch.zeros(out)))


@pytest.mark.parametrize("kw, err, what", [
    (dict(norm_weight=None), TypeError, "norm_weight"),
    (dict(residual=bf(4, 33)), TypeError, "rows of"),
    (dict(post_weight=bf(33)), TypeError, "norm weights"),
    (dict(next_weight=bf(31)), TypeError, "norm weights"),
    (dict(post_weight=bf(32), next_weight=torch.zeros(32)), TypeError, "norm weights"),
    (dict(gate=bf(4)), ValueError, "gate of shape"),
    (dict(gate=torch.zeros(32)), TypeError, "gate of"),
    (dict(residual_scale="half"), ValueError, "float"),
    (dict(shared_expert=expert(inner=64)), ValueError, "shared_expert"),
    (dict(shared_expert=expert(up=128)), ValueError, "shared_expert"),
    (dict(shared_expert=expert(hidden=48)), ValueError, "shared_expert"),
    (dict(shared_expert=expert(out=48)), ValueError, "shared_expert"),
    (dict(shared_expert=expert(inner=0)), ValueError, "shared_expert"),
    (dict(shared_expert=expert(inner=131072)), ValueError, "shared_expert"),
    (dict(shared_expert=expert(dtype=torch.uint8)), TypeError, "int8"),
    (dict(shared_expert=(expert()[0], (expert()[1][0], torch.zeros(31)))), TypeError, "down: fp32 scales"),
    (dict(shared_expert=expert(), activation_clamp=-1.0), ValueError, "activation_clamp"),
    (dict(shared_expert=expert()), RuntimeError, "GPU"),
])
def test_refusals_come_before_the_layer(kw, err, what, monkeypatch):
    from hopper_megamoe_basedondeepgemm_amd import block as module
    monkeypatch.setattr(module, "mxfp4_mega_moe_from_bf16", lambda *a, **k: pytest.fail("the layer has run"))
    with pytest.raises(err, match=what):
        block(**kw)


def test_refusals_do_not_wait_for_the_first_norm(monkeypatch):
    from hopper_megamoe_basedondeepgemm_amd import block as module
    monkeypatch.setattr(module, "_norm", lambda *a, **k: pytest.fail("a norm has run"))
    for kw in (dict(post_weight=bf(33)), dict(gate=bf(4)), dict(shared_expert=expert(out=48)), dict(shared_expert=expert())):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            block(**kw)
