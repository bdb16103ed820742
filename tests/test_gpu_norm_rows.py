"""The backward pass of rms_norm_residual where a workgroup takes several rows.

A call gets at most 4096 workgroups up to hidden 512, 2048 up to 1024, 1024 up to 2048, 512 up to 4096 and 256
beyond; with more rows a workgroup requests its next row ahead, takes its two sets of LDS sums in turn and
carries the column sums over its rows. Formulas and tolerances are those of test_gpu_norm."""
import pytest
import torch

from tests.gpu_common import need_gpu
from tests.test_gpu_norm import check_forward, close, make

pytestmark = pytest.mark.gpu

# (the last round of rows is uneven in all; the widths before and behind each limit, and off 8 elements)
SHAPES = [(9001, 64), (4500, 100), (2100, 1000), (2300, 1024), (1030, 2047), (1100, 2880), (1030, 4096), (700, 5001), (600, 8192),
          (300, 9000), (300, 16384), (259, 10001)]
# post, pre, gate, residual, sigmoid, scale, fp32 weights: 0 to 2 reductions a row
FORMS = [(0, 0, "channel", 1, False, 2.0, False), (0, 1, "none", 1, False, 1.0, False), (0, 0, "token", 1, True, 0.5, False),
         (1, 0, "full", 1, False, 1.0, True), (1, 1, "channel", 1, True, 0.22, False), (1, 1, "token", 1, False, 1.0, True),
         (1, 1, "full", 0, True, -0.5, False)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gradients_of_many_rows(T, H, dtype):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    from hopper_megamoe_basedondeepgemm_amd import _lib
    assert _lib.load().dgm_rms_norm_residual_groups(T, H) < T
    for post, pre, gate, residual, sigmoid, s, f32 in FORMS:
        x, r, w1, w2, gt = make(T, H, dtype, torch.float32 if f32 else dtype, post, pre, gate, residual, seed=T + H)
        ins = dict(x=x, residual=r, post=w1, pre=w2, gate=gt)
        leaves = {k: v.requires_grad_() for k, v in ins.items() if v is not None}
        got_r, got_h = dgm.rms_norm_residual(x, r, w1, w2, gt, sigmoid, s)
        f = check_forward(x, r, w1, w2, gt, sigmoid, s, got_r, got_h)
        dr = torch.randn_like(got_r)
        dh = None if got_h is None else torch.randn_like(got_h)
        outs, douts = ([got_r, got_h], [dr, dh]) if got_h is not None else ([got_r], [dr])
        grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), douts)))
        want = f.grads(dr, dh)
        if r is None:
            del want["residual"]
        assert set(want) == set(grads)
        for k, (v, m) in want.items():
            assert grads[k].shape == ins[k].shape and grads[k].dtype == ins[k].dtype
            over = T if v.dim() == 1 else H if v.shape != f.t.shape else 0
            close(grads[k], v, m, 256 + over)
