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
    return dgm.mega_moe_block(bf(4, 32), bf(32), bf(4, 32), None, None, sym_buffer or buffer(), **kw)


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
    monkeypatch.setattr(module, "rms_norm_residual", lambda x, residual=None, *a, **kw: (x, x))
    block(cumulative_local_expert_recv_stats=1, activation_clamp=2.0, force_balanced=True, token_offset=3, phase_stamps=4,
          one_launch=False)
    assert seen == dict(stats=1, clamp=2.0, balanced=True, offset=3, stamps=4, one=False)
