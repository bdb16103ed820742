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
