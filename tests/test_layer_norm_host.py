"""layer_norm_residual: what is refused before any GPU work, and what autograd is told (CPU)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import hopper_megamoe_basedondeepgemm_amd as dgm
from hopper_megamoe_basedondeepgemm_amd import _lib
from tests.no_launch_rows import launches  # noqa: F401


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_struct_sizes():
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert _lib.load().dgm_layer_norm_struct_sizes(ctypes.byref(a), ctypes.byref(b)) == 0
    assert a.value == ctypes.sizeof(_lib.LayerNormArgs) and b.value == ctypes.sizeof(_lib.LayerNormGradArgs)


@pytest.mark.parametrize("x, kw, err, what", [
    (bf(32), {}, TypeError, "x must be"),
    (torch.zeros((4, 32), dtype=torch.float64), {}, TypeError, "x must be"),
    (bf(4, 0), {}, ValueError, "hidden"),
    (bf(4, 16385), {}, ValueError, "hidden"),
    (bf(1, 8).expand(1 << 22, 8), {}, ValueError, "tokens"),
    (bf(4, 32), dict(residual=bf(4, 33)), TypeError, "rows of"),
    (bf(4, 32), dict(residual=torch.zeros(4, 32)), TypeError, "rows of"),
    (bf(4, 32), dict(weight=bf(33)), TypeError, "weight and bias"),
    (bf(4, 32), dict(weight=bf(1, 32)), TypeError, "weight and bias"),
    (bf(4, 32), dict(bias=torch.zeros(32, dtype=torch.float16)), TypeError, "weight and bias"),
    (bf(4, 32), dict(weight=bf(32), bias=torch.zeros(32)), TypeError, "weight and bias"),
    (bf(4, 32), dict(quant="int8"), ValueError, "quant"),
    (torch.zeros(4, 32), dict(quant="mxfp4"), ValueError, "bf16"),
    (bf(4, 32), dict(out=bf(32, 4).t()), ValueError, "contiguous"),
    (bf(4, 32), dict(residual_out=bf(1, 32).expand(4, 32)), ValueError, "overlap"),
    (bf(4, 32), dict(out=bf(4, 33)), TypeError, "rows of"),
    (bf(4, 32), dict(residual_scale="half"), (ValueError, RuntimeError), "float|GPU"),
    (bf(4, 32), {}, RuntimeError, "GPU"),
])
def test_refusals(x, kw, err, what):
    with pytest.raises(err, match=what):
        dgm.layer_norm_residual(x, **kw)


def test_backward_refusals():
    x, r, w, b, st = bf(4, 32), bf(4, 32), bf(32), bf(32), torch.zeros(4)
    call = lambda d_r=x, d_h=x, x=x, r=r, mean=st, rstd=st, w=w, b=b: dgm.layer_norm_residual_backward(d_r, d_h, x, r, mean, rstd, w, b)
    for kw, err, what in ((dict(d_r=bf(4, 31)), TypeError, "gradient rows"), (dict(d_h=torch.zeros(4, 32)), TypeError, "gradient rows"),
                          (dict(mean=None), ValueError, "mean and rstd"), (dict(rstd=torch.zeros(5)), ValueError, "mean and rstd"),
                          (dict(rstd=bf(4)), ValueError, "mean and rstd"), (dict(mean=torch.zeros(8)[::2]), ValueError, "mean and rstd"),
                          (dict(w=bf(31)), TypeError, "weight and bias"), (dict(), RuntimeError, "GPU")):
        with pytest.raises(err, match=what):
            call(**kw)


def args():
    return dict(x=torch.randn(4, 16), residual=torch.randn(4, 16), weight=torch.ones(16), bias=torch.zeros(16))


@pytest.mark.parametrize("name", ["x", "residual", "weight", "bias"])
def test_tangents_are_refused(launches, name):  # noqa: F811
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
    a = args()
    with forward_ad.dual_level():
        dgm.layer_norm_residual(**a)
        launches.calls.clear()
        d = {**a, name: dual(a[name])}
        for call in (dgm.layer_norm_residual, dgm.layer_norm_residual_forward):
            with pytest.raises(RuntimeError, match="tangent"):
                call(**d)
        with pytest.raises(RuntimeError, match="tangent"):
            dgm.layer_norm_residual_backward(torch.ones(4, 16), None, d["x"], d["residual"], torch.ones(4), torch.ones(4), d["weight"], d["bias"])
        for out in ("residual_out", "out"):
            with pytest.raises(RuntimeError, match="tangent"):
                dgm.layer_norm_residual(**a, **{out: dual(torch.zeros(4, 16))})
        assert not launches.calls
        leaf = a["x"].requires_grad_()
        r, h = dgm.layer_norm_residual(**a)
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad((r, h), leaf, (dual(torch.ones(4, 16)), torch.ones(4, 16)))


def saved():
    leaf = torch.randn(4, 16, requires_grad=True)
    mid = leaf * 2
    return leaf, mid, (mid * mid).sum()


@pytest.mark.parametrize("name", ["residual_out", "out"])
def test_rows_that_a_graph_has_saved(launches, name):  # noqa: F811
    leaf, mid, loss = saved()
    with torch.no_grad():
        dgm.layer_norm_residual(torch.randn(2, 16), **{name: mid[1:3]})
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, leaf)


def test_outputs(launches):  # noqa: F811
    """Over an input's own rows, not over parts of them or one another; not where a gradient is asked for."""
    x, r = torch.randn(6, 16), torch.randn(6, 16)
    assert dgm.layer_norm_residual(x, r, residual_out=r, out=x)[0] is r
    dgm.layer_norm_residual(x, r, residual_out=x, out=r)
    launches.calls.clear()
    for kw in (dict(x=x[:4], out=x[1:5]), dict(x=x[:4], residual=r[:4], residual_out=r[2:]), dict(x=x, residual_out=r, out=r)):
        with pytest.raises(ValueError, match="overlap"):
            dgm.layer_norm_residual(**kw)
    w = torch.ones(32)
    with pytest.raises(ValueError, match="overlap"):
        dgm.layer_norm_residual(torch.randn(1, 16), weight=w[4:20], out=w[:16].view(1, 16))
    for kw in (dict(out=torch.zeros(6, 16)), dict(residual_out=torch.zeros(6, 16))):
        with pytest.raises(ValueError, match="no gradient"):
            dgm.layer_norm_residual(x.clone().requires_grad_(), **kw)
    with pytest.raises(ValueError, match="no gradient"):
        dgm.layer_norm_residual(x, out=torch.zeros(6, 16, requires_grad=True))
    with pytest.raises(ValueError, match="no gradient"):
        dgm.layer_norm_residual(bf(4, 32).requires_grad_(), quant="mxfp4")
    assert not launches.calls
    x = torch.randn(4, 16)
    launches.status = -1
    with pytest.raises(RuntimeError, match="dgm error"):
        dgm.layer_norm_residual(x, out=x)
    assert x._version == 0


def norm(change, **kw):
    x = torch.randn(6, 16, requires_grad=True)
    a = dict(residual=torch.randn(6, 16, requires_grad=True), weight=torch.ones(16), bias=torch.ones(16))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t.clone())):
        r, h = dgm.layer_norm_residual(x, **{**a, **kw})
    torch.autograd.grad((r, h), x, (torch.ones_like(r), torch.ones_like(h)))


@pytest.mark.parametrize("change", [
    lambda t: t.bfloat16() if t.shape == (6, 16) else t,
    lambda t: t[:3] if t.shape == (6, 16) else t,
    lambda t: t[:, :8] if t.shape == (6, 16) else t,
    lambda t: t[:8] if t.shape == (16,) else t,
    lambda t: t.half() if t.shape == (16,) else t,
    lambda t: t.half() if t.shape == (2, 6) else t,
    lambda t: t[:1] if t.shape == (2, 6) else t,
    lambda t: t[:, :3] if t.shape == (2, 6) else t,
])
def test_saved_tensors_that_come_back_changed(launches, change):  # noqa: F811
    norm(lambda t: t)
    assert launches.calls == ["dgm_layer_norm_residual", "dgm_layer_norm_residual_backward"]
    launches.calls.clear()
    with pytest.raises((TypeError, ValueError)):
        norm(change)
    assert launches.calls == ["dgm_layer_norm_residual"]


def test_r_is_x_where_nothing_changes_it(launches):  # noqa: F811
    x = torch.randn(4, 16)
    assert dgm.layer_norm_residual(x)[0] is x
    assert dgm.layer_norm_residual(x, residual_scale=2.0)[0] is not x
    x.requires_grad_()
    r, h = dgm.layer_norm_residual(x)
    assert r.data_ptr() == x.data_ptr() and r.requires_grad
    torch.autograd.grad((r, h), x, (torch.ones(4, 16), torch.ones(4, 16)))
    assert launches.calls[-1] == "dgm_layer_norm_residual_backward"


def test_c_entry_refusals():
    lib, p = _lib.load(), 4096          # (never dereferenced: refused first)
    base = dict(x=p, h=p, rows=4, hidden=64, x_stride=64, h_stride=64, eps=1e-5)
    for kw, what in ((dict(dtype=3), b"dtype"), (dict(rows=-1), b"rows"), (dict(rows=1 << 22), b"rows"), (dict(hidden=0), b"hidden"),
                     (dict(hidden=16385), b"hidden"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(x=None), b"null x"),
                     (dict(codes=p), b"their scales"), (dict(mean=p), b"mean with rstd"), (dict(codes=p, scales=p, dtype=1), b"MXFP4 rows"),
                     (dict(codes=p, scales=p, x=p + 2), b"MXFP4 rows"), (dict(codes=p, scales=p, hidden=63), b"MXFP4 rows")):
        st = lib.dgm_layer_norm_residual(ctypes.byref(_lib.LayerNormArgs(**{**base, **kw})), None)
        assert st == -1 and what in lib.dgm_last_error(), (kw, lib.dgm_last_error())
    assert lib.dgm_layer_norm_residual(ctypes.byref(_lib.LayerNormArgs(**{**base, "rows": 0, "x": None})), None) == 0
    assert lib.dgm_layer_norm_residual(None, None) == -1
    forward = dict(**base, weight=p, bias=p, residual=p, mean=p, rstd=p)
    grad = dict(d_h=p, d_x=p, d_weight=p, workspace=p, workspace_bytes=1 << 30)
    for fkw, kw, what in ((dict(mean=None), {}, b"mean and rstd"), (dict(residual=None), dict(d_residual=p), b"without a residual"),
                          (dict(weight=None), {}, b"without its weight"), (dict(bias=None), dict(d_bias=p), b"without its bias"),
                          ({}, dict(workspace=None), b"workspace"), ({}, dict(workspace=p + 4), b"workspace"), ({}, dict(workspace_bytes=64), b"workspace")):
        a = _lib.LayerNormGradArgs(forward=_lib.LayerNormArgs(**{**forward, **fkw}), **{**grad, **kw})
        st = lib.dgm_layer_norm_residual_backward(ctypes.byref(a), None)
        assert st == -1 and what in lib.dgm_last_error(), (fkw, kw, lib.dgm_last_error())
    assert lib.dgm_layer_norm_residual_backward(None, None) == -1
