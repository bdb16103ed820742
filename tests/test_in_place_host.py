"""Outputs that a caller gives (CPU, launches left out): autograd learns of the write, or the call is refused."""
import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm
from tests.no_launch import no_launch  # noqa: F401


def saved():
    """(a tensor that an earlier graph needs in its backward pass, that graph's result)"""
    leaf = torch.randn(4, 16, requires_grad=True)
    mid = leaf * 2
    return leaf, mid, (mid * mid).sum()


@pytest.mark.parametrize("name", ["residual_out", "out"])
@pytest.mark.parametrize("part", [False, True])
def test_norm_rows_that_a_graph_has_saved(no_launch, name, part):  # noqa: F811
    leaf, mid, loss = saved()
    with torch.no_grad():
        rows = mid[1:3] if part else mid
        dgm.rms_norm_residual(torch.randn(rows.shape), pre_weight=torch.ones(16), **{name: rows})
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, leaf)


@pytest.mark.parametrize("add", [False, True])
def test_product_rows_that_a_graph_has_saved(no_launch, add):  # noqa: F811
    leaf, mid, loss = saved()
    a, b = (torch.zeros((4, 32), dtype=torch.int8), torch.ones(4)), (torch.zeros((16, 32), dtype=torch.int8), torch.ones(16))
    with torch.no_grad():
        dgm.int8_gemm_nt(a, b, mid, c=mid if add else None)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, leaf)


def test_under_inference_mode(no_launch):  # noqa: F811
    with torch.inference_mode():
        x = torch.randn(4, 16)
        dgm.rms_norm_residual(x, pre_weight=torch.ones(16), out=x, residual_out=torch.empty(4, 16))
        dgm.int8_gemm_nt((torch.zeros((4, 32), dtype=torch.int8), torch.ones(4)),
                         (torch.zeros((16, 32), dtype=torch.int8), torch.ones(16)), x)
    assert len(no_launch.calls) == 2


def test_nothing_written_is_nothing_changed(no_launch):  # noqa: F811
    """A call that is refused, or has no rows, leaves the version."""
    x = torch.randn(4, 16)
    with pytest.raises(ValueError, match="overlaps an input"):
        dgm.rms_norm_residual(x[:3], pre_weight=torch.ones(16), out=x[1:])
    dgm.rms_norm_residual(x[:0], pre_weight=torch.ones(16), out=x[:0])
    no_launch.status = -1
    with pytest.raises(RuntimeError, match="dgm error"):
        dgm.rms_norm_residual(torch.randn(4, 16), pre_weight=torch.ones(16), out=x)
    assert x._version == 0


@pytest.mark.parametrize("name", ["residual_out", "out"])
def test_an_output_that_asks_for_a_gradient(no_launch, name):  # noqa: F811
    x, w = torch.randn(4, 16), torch.ones(16)
    for rows in (torch.zeros(4, 16, requires_grad=True), torch.zeros(4, 16, requires_grad=True) * 1):
        with pytest.raises(ValueError, match="no gradient"):
            dgm.rms_norm_residual(x, pre_weight=w, **{name: rows})
        assert not no_launch.calls
        with torch.no_grad():
            dgm.rms_norm_residual(x, pre_weight=w, **{name: rows})
        no_launch.calls.clear()


@pytest.mark.parametrize("which,scales,apart", [
    ("a", slice(46, 50), True), ("a", slice(47, 51), False), ("a", slice(113, 117), False), ("a", slice(114, 118), True),
    ("a", slice(40, 47, 2), True), ("a", slice(45, 52, 2), False), ("b", slice(34, 50), True), ("b", slice(35, 51), False),
    ("b", slice(113, 129), False), ("b", slice(114, 130), True), ("b", slice(20, 51, 2), False), ("b", slice(18, 49, 2), True)])
def test_a_product_over_its_own_scales(no_launch, which, scales, apart):  # noqa: F811
    """d is written while other workgroups still read the scales."""
    memory = torch.ones(200)
    d, mine = memory[50:114].view(4, 16), memory[scales]
    a = torch.zeros((4, 32), dtype=torch.int8), mine if which == "a" else torch.ones(4)
    b = torch.zeros((16, 32), dtype=torch.int8), mine if which == "b" else torch.ones(16)
    if apart:
        dgm.int8_gemm_nt(a, b, d)
    else:
        with pytest.raises(ValueError, match="d overlaps"):
            dgm.int8_gemm_nt(a, b, d)
    assert len(no_launch.calls) == apart
