"""layer_norm_residual over its inputs' own rows, at lengths whose last elements are read by two threads of different
waves (a row of 513 elements ends one behind a wave's)."""
import pytest
import torch

from tests.gpu_common import need_gpu
from tests.test_gpu_layer_norm import DT, Form, close, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H", [9, 511, 513, 519, 1025, 1027, 2055, 4097, 5001, 8193, 8199, 12345, 16383])
def test_outputs_over_their_inputs(H, dtype):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w, b, *_ = make(300, H, dtype, dtype, seed=H)
    f = Form(x, r, w, b, 0.5)
    want = dgm.layer_norm_residual(x, r, w, b, 0.5)
    close(want[0], f.t, f.t_mag, 128)
    close(want[1], f.h, f.h_mag, 128)

    def within(t):
        big = torch.full((302, H + 12), 5.0, dtype=dtype, device="cuda")
        view = big[1:301, 3:3 + H]
        view.copy_(t)
        return view, big
    for which in ("residual, x", "x, residual", "x, none", "none, residual", "residual, none", "none, x"):
        (xs, all_x), (rs, all_r) = within(x), within(r)
        named = {"x": xs, "residual": rs, "none": None}
        r_out, out = (named[n] for n in which.split(", "))
        got = dgm.layer_norm_residual(xs, rs, w, b, 0.5, residual_out=r_out, out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), which
        assert (r_out is None or got[0] is r_out) and (out is None or got[1] is out)
        for view, big, t in ((xs, all_x, x), (rs, all_r, r)):
            if view is not r_out and view is not out:
                assert torch.equal(view, t)
            view.fill_(5.0)
            assert bool((big == 5.0).all()), which
