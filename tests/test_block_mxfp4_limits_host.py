"""mega_moe_block with an MXFP4 dense expert: a product that is refused is refused before the layer counts its tokens (CPU)."""
import types

import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm
from hopper_megamoe_basedondeepgemm_amd import block as module


def weights(m, k):
    return torch.zeros((1, 16 * (k // 32)), dtype=torch.uint8).expand(m, -1), torch.zeros((1, k // 32), dtype=torch.uint8).expand(m, -1)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("tokens, hidden, inner, fits", [
    (1 << 21, 16384, 32, False),                   # the down product: 2^15 x 2^8 tiles
    ((1 << 21) - 64, 16384, 32, True),
    (1 << 20, 64, 16384, False),                   # gate and up: 2^14 x 2^9
    ((1 << 20) - 64, 64, 16384, True),
])
def test_both_products_are_checked_first(norm, tokens, hidden, inner, fits, monkeypatch):
    class Reached(Exception):
        pass

    def stop(*tensors):
        raise Reached
    monkeypatch.setattr(module._lib, "require_one_device", stop)           # (the last check before the first launch)
    buffer = types.SimpleNamespace(hidden=hidden, num_experts=4, num_local_experts=4, ep_size=1)
    x, w = torch.zeros((1, hidden), dtype=torch.bfloat16).expand(tokens, hidden), torch.zeros(hidden, dtype=torch.bfloat16)
    with pytest.raises(Reached if fits else ValueError, match=None if fits else "2.23"):
        dgm.mega_moe_block(x, w, torch.zeros((4, hidden), dtype=torch.bfloat16), None, None, buffer, norm=norm,
                           shared_expert=(weights(2 * inner, hidden), weights(hidden, inner)))
