"""mxfp4_quantize, mxfp4_gemm_nt and mxfp4_linear: what is refused before any GPU work, and what autograd is told (CPU)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import hopper_megamoe_basedondeepgemm_amd as dgm
from hopper_megamoe_basedondeepgemm_amd import _lib
from tests.no_launch_rows import launches  # noqa: F401

U8 = torch.uint8


def rows(m, k):
    return torch.zeros((m, k // 2), dtype=U8), torch.zeros((m, k // 32), dtype=U8)


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_struct_sizes():
    a = ctypes.c_size_t(0)
    for name, struct in (("quant", _lib.Mxfp4QuantArgs), ("gemm", _lib.Mxfp4GemmArgs), ("linear", _lib.Mxfp4LinearArgs)):
        assert getattr(_lib.load(), f"dgm_mxfp4_{name}_struct_size")(ctypes.byref(a)) == 0 and a.value == ctypes.sizeof(struct)


@pytest.mark.parametrize("x, kw, err, what", [
    (torch.zeros((4, 32), dtype=torch.float64), {}, TypeError, "x must be"),
    (torch.zeros((4, 32), dtype=U8), {}, TypeError, "x must be"),
    (bf(32), {}, TypeError, "x must be"),
    (bf(2, 4, 32), {}, TypeError, "x must be"),
    (bf(1, 1).expand(1 << 24, 1), {}, ValueError, "2.24"),
    (bf(1, 1).expand(1, 1 << 24), {}, ValueError, "2.24"),
    (bf(4, 32), dict(amax_floor=-1.0), ValueError, "amax_floor"),
    (bf(4, 32), dict(amax_floor=float("nan")), ValueError, "amax_floor"),
    (bf(4, 32), dict(amax_floor=float("inf")), ValueError, "amax_floor"),
    (bf(4, 32).requires_grad_(), {}, RuntimeError, "no gradient"),
    (bf(4, 32), {}, RuntimeError, "GPU"),
])
def test_quantize_refusals(x, kw, err, what):
    for call in (dgm.mxfp4_quantize, dgm.mxfp4_quantize_both):
        with pytest.raises(err, match=what):
            call(x, **kw)


@pytest.mark.parametrize("a, b, d, kw, err, what", [
    ((bf(4, 32), torch.zeros(4, 2)), rows(8, 64), bf(4, 8), {}, TypeError, "a: uint8 codes"),
    ((rows(4, 64)[0], torch.zeros(4, 2)), rows(8, 64), bf(4, 8), {}, TypeError, "a: uint8 scales"),
    (rows(4, 64), (rows(8, 64)[0], rows(7, 64)[1]), bf(4, 8), {}, TypeError, "b: uint8 scales"),
    (rows(4, 64), (rows(8, 64)[0], rows(8, 96)[1]), bf(4, 8), {}, TypeError, "b: uint8 scales"),
    (rows(4, 64), (torch.zeros((8, 24), dtype=U8), torch.zeros((8, 2), dtype=U8)), bf(4, 8), {}, TypeError, "b: uint8 scales"),
    ((rows(4, 64)[0], torch.zeros(4, dtype=U8)), rows(8, 64), bf(4, 8), {}, TypeError, "a: uint8 scales"),
    (rows(4, 64), rows(8, 96), bf(4, 8), {}, ValueError, "k of a"),
    (rows(4, 0), rows(8, 0), bf(4, 8), {}, ValueError, "k of a"),
    (rows(4, 64), rows(8, 64), bf(4, 9), {}, TypeError, "d: bf16"),
    (rows(4, 64), rows(8, 64), bf(32), {}, TypeError, "d: bf16"),
    (rows(4, 64), rows(8, 64), torch.zeros((4, 8), dtype=torch.float64), {}, TypeError, "d: bf16"),
    (rows(4, 64), rows(8, 64), bf(8, 4).t(), {}, ValueError, "d: rows"),
    (rows(4, 64), rows(8, 64), bf(1, 8).expand(4, 8), {}, ValueError, "d: rows"),
    (rows(4, 64), rows(8, 64), bf(4, 8), dict(c=torch.zeros(4, 8)), TypeError, "c: "),
    (rows(4, 64), rows(8, 64), bf(4, 8), dict(c=bf(4)), TypeError, "c: "),
    (rows(4, 64), rows(8, 64), bf(4, 8), dict(activation="gelu"), ValueError, "activation"),
    (rows(4, 64), rows(7, 64), bf(4, 3), dict(activation="swiglu"), ValueError, "swiglu"),
    (rows(4, 64), rows(8, 64), bf(4, 4), dict(activation="swiglu", c=bf(4, 4)), ValueError, "swiglu"),
    (rows(4, 64), rows(8, 64), bf(4, 4), dict(activation="swiglu", activation_clamp=-1.0), ValueError, "activation_clamp"),
    (rows(4, 64), rows(8, 64), bf(4, 4), dict(activation="swiglu", activation_clamp=float("nan")), ValueError, "activation_clamp"),
    (rows(4, 64), rows(8, 64), bf(4, 8).requires_grad_(), {}, RuntimeError, "no gradient"),
    (rows(4, 64), rows(8, 64), bf(4, 8), dict(c=bf(8).requires_grad_()), RuntimeError, "no gradient"),
    (rows(4, 64), rows(8, 64), bf(4, 8), {}, RuntimeError, "GPU"),
])
def test_gemm_refusals(a, b, d, kw, err, what):
    with pytest.raises(err, match=what):
        dgm.mxfp4_gemm_nt(a, b, d, **kw)


def test_gemm_sizes(launches):  # noqa: F811
    big = tuple(t.expand(1 << 24, -1) for t in rows(1, 32))
    with pytest.raises(ValueError, match="below 2.24"):
        dgm.mxfp4_gemm_nt(big, rows(8, 32), bf(1, 8).expand(1 << 24, 8))
    many = tuple(t.expand(1 << 21, -1) for t in rows(1, 32))
    with pytest.raises(ValueError, match="2.23"):
        dgm.mxfp4_gemm_nt(many, many, bf(1, 1).expand(1 << 21, 1 << 21))
    d = bf(0, 8)
    assert dgm.mxfp4_gemm_nt(rows(0, 64), rows(8, 64), d) is d
    assert not launches.calls


@pytest.mark.parametrize("which,part,apart", [
    ("a", slice(0, 64), True), ("a", slice(208, 272), False), ("a", slice(200, 264), True), ("b", slice(0, 512), False), ("b", slice(192, 704), False),
    ("sa", slice(124, 128), True), ("sa", slice(126, 130), False), ("sb", slice(383, 399), False), ("sb", slice(384, 400), True)])
def test_a_product_over_its_own_operands(launches, which, part, apart):  # noqa: F811
    """d is written while other workgroups still read. (Codes off 16 bytes are read from a copy.)"""
    memory = torch.zeros(1024, dtype=U8)
    d = memory[128:384].view(torch.float32).view(4, 16)
    t = dict(a=torch.zeros((4, 16), dtype=U8), sa=torch.zeros((4, 1), dtype=U8), b=torch.zeros((16, 16), dtype=U8), sb=torch.zeros((16, 1), dtype=U8))
    mine = memory[part]
    t[which] = mine.view(t[which].shape[0], -1)[:, :t[which].shape[1]]
    run = lambda: dgm.mxfp4_gemm_nt((t["a"], t["sa"]), (t["b"], t["sb"]), d)
    if apart:
        run()
    else:
        with pytest.raises(ValueError, match="d overlaps"):
            run()
    assert len(launches.calls) == apart


def test_c_over_d(launches):  # noqa: F811
    d = torch.zeros(8, 32)
    a, b = rows(4, 64), rows(32, 64)
    dgm.mxfp4_gemm_nt(a, b, d[:4], c=d[:4])
    dgm.mxfp4_gemm_nt(a, b, d[:4], c=d[4:])
    for c in (d[1:5], d[0]):
        with pytest.raises(ValueError, match="c overlaps"):
            dgm.mxfp4_gemm_nt(a, b, d[:4], c=c)
    assert len(launches.calls) == 2


@pytest.mark.parametrize("x, w, err, what", [
    (bf(4, 32), bf(8, 33), TypeError, "weight must"),
    (bf(4, 32), bf(32), TypeError, "weight must"),
    (bf(4, 32), torch.zeros((8, 32), dtype=torch.int8), TypeError, "weight must"),
    (torch.zeros((4, 32), dtype=torch.float64), bf(8, 32), TypeError, "x must"),
    (bf(4, 0), bf(8, 0), ValueError, "no feature"),
    (bf(4, 8), bf(0, 8), ValueError, "no feature"),
    (bf(1, 1).expand(1 << 21, 1), bf(1, 1).expand(1 << 21, 1), ValueError, "2.23"),
    (bf(4, 32), bf(8, 32), RuntimeError, "GPU"),
])
def test_linear_refusals(x, w, err, what):
    for call in (dgm.mxfp4_linear, dgm.mxfp4_linear_forward):
        with pytest.raises(err, match=what):
            call(x, w)


def test_linear_backward_refusals():
    xt, wt = rows(32, 32), rows(32, 64)          # columns of x [4, 32] and of the weight [40, 32]
    call = lambda d_y=bf(4, 40), xt=xt, wt=wt, xs=(4, 32), ws=(40, 32), **kw: dgm.mxfp4_linear_backward(d_y, xt, wt, xs, ws, **kw)
    for kw, err, what in ((dict(d_y=bf(4, 41)), TypeError, "d_y"), (dict(d_y=bf(5, 40)), TypeError, "d_y"),
                          (dict(d_y=torch.zeros(4, 40, dtype=torch.float64)), TypeError, "bf16, fp16"),
                          (dict(weight_dtype=torch.int8), TypeError, "bf16, fp16"), (dict(xs=(4, 33)), ValueError, "tokens"),
                          (dict(ws=(40,)), ValueError, "tokens"), (dict(xt=None), ValueError, "x_columns"),
                          (dict(wt=None), ValueError, "weight_columns"), (dict(xt=rows(33, 32)), ValueError, "x_columns"),
                          (dict(xt=(xt[0], xt[1].int())), ValueError, "x_columns"), (dict(wt=rows(32, 32)), ValueError, "weight_columns"),
                          (dict(wt=(wt[0], xt[1])), ValueError, "weight_columns"), (dict(), RuntimeError, "GPU"),
                          (dict(xt=None, needs=(True, False)), RuntimeError, "GPU"), (dict(wt=None, needs=(False, True)), RuntimeError, "GPU")):
        with pytest.raises(err, match=what):
            call(**kw)


def test_tangents_are_refused(launches):  # noqa: F811
    x, w, d, dy = torch.randn(4, 32), torch.randn(8, 32), torch.zeros(4, 8), torch.randn(4, 8)
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
    _, xt, wt = dgm.mxfp4_linear_forward(x, w)
    launches.calls.clear()
    with forward_ad.dual_level():
        for call in (lambda: dgm.mxfp4_quantize(dual(x)), lambda: dgm.mxfp4_quantize_both(dual(x)), lambda: dgm.mxfp4_linear(dual(x), w),
                     lambda: dgm.mxfp4_linear(x, dual(w)), lambda: dgm.mxfp4_linear_forward(dual(x), w),
                     lambda: dgm.mxfp4_linear_backward(dual(dy), xt, wt, x.shape, w.shape),
                     lambda: dgm.mxfp4_gemm_nt(rows(4, 64), rows(8, 64), dual(d)), lambda: dgm.mxfp4_gemm_nt(rows(4, 64), rows(8, 64), d, c=dual(dy))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert not launches.calls
        y = dgm.mxfp4_linear(x.requires_grad_(), w)
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(y, x, dual(dy))


def test_rows_that_a_graph_has_saved(launches):  # noqa: F811
    leaf = torch.randn(4, 8, requires_grad=True)
    mid = leaf * 2
    loss = (mid * mid).sum()
    with torch.no_grad():
        dgm.mxfp4_gemm_nt(rows(4, 64), rows(8, 64), mid)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, leaf)


def linear(change, needs=(True, True)):
    x, w = torch.randn(6, 40, requires_grad=needs[0]), torch.randn(70, 40, requires_grad=needs[1])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t.clone())):
        y = dgm.mxfp4_linear(x, w)
    return torch.autograd.grad(y, [t for t in (x, w) if t.requires_grad], torch.ones_like(y))


@pytest.mark.parametrize("change", [lambda t: t.to(torch.int8), lambda t: t[:-1], lambda t: t[:0], lambda t: t.view(2, -1)])
def test_saved_columns_that_come_back_changed(launches, change):  # noqa: F811
    got = linear(lambda t: t)
    assert [tuple(g.shape) for g in got] == [(6, 40), (70, 40)] and launches.calls == ["dgm_mxfp4_linear", "dgm_mxfp4_linear_backward"]
    for needs in ((True, True), (True, False), (False, True)):
        launches.calls.clear()
        with pytest.raises(ValueError, match="saved columns"):
            linear(change, needs)
        assert launches.calls == ["dgm_mxfp4_linear"]


def test_no_tokens(launches):  # noqa: F811
    x, w = torch.zeros(0, 64, requires_grad=True), torch.ones(32, 64, requires_grad=True)
    y = dgm.mxfp4_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 64) and not bool(dw.any()) and launches.calls == ["dgm_mxfp4_linear"]


def test_c_entry_refusals():
    lib, p = _lib.load(), 4096          # (never dereferenced: refused first)
    quant = dict(x=p, codes=p, scales=p, rows=4, cols=64, x_stride=64)
    for kw, what in ((dict(dtype=3), b"dtype"), (dict(rows=-1), b"below 2^24"), (dict(cols=1 << 24), b"below 2^24"), (dict(x_stride=-1), b"stride"),
                     (dict(amax_floor=-1.0), b"amax_floor"), (dict(amax_floor=float("nan")), b"amax_floor"), (dict(scales=None), b"their scales"),
                     (dict(t_codes=p), b"their scales"), (dict(x=None), b"null pointer"), (dict(codes=None, scales=None), b"null pointer"),
                     (dict(codes=p + 8), b"16 bytes"), (dict(rows=(1 << 24) - 1, cols=(1 << 24) - 1), b"2^32 threads")):
        st = lib.dgm_mxfp4_quantize(ctypes.byref(_lib.Mxfp4QuantArgs(**{**quant, **kw})), None)
        assert st == -1 and what in lib.dgm_last_error(), (kw, lib.dgm_last_error())
    assert lib.dgm_mxfp4_quantize(ctypes.byref(_lib.Mxfp4QuantArgs(**{**quant, "rows": 0})), None) == 0
    assert lib.dgm_mxfp4_quantize(None, None) == -1
    gemm = dict(a=p, sfa=p, b=p, sfb=p, d=p, m=4, n=8, k=64, a_stride=32, b_stride=32, sfa_stride=2, sfb_stride=2, d_stride=8)
    for kw, what in ((dict(dtype=3), b"dtype"), (dict(k=0), b"multiple of 32"), (dict(k=48), b"multiple of 32"), (dict(k=1 << 24), b"multiple of 32"),
                     (dict(m=-1), b"below 2^24"), (dict(n=1 << 24), b"below 2^24"), (dict(swiglu=1, c=p), b"SwiGLU"), (dict(swiglu=1, n=7), b"SwiGLU"),
                     (dict(sfa_stride=-1), b"strides"), (dict(a_stride=40), b"16 bytes"), (dict(b=p + 8), b"16 bytes"),
                     (dict(a_stride=1 << 23), b"2^23 bytes apart"), (dict(d=None), b"null pointer"), (dict(sfb=None), b"null pointer"),
                     (dict(m=1 << 21, n=1 << 21), b"below 2^23")):
        st = lib.dgm_mxfp4_gemm_nt(ctypes.byref(_lib.Mxfp4GemmArgs(**{**gemm, **kw})), None)
        assert st == -1 and what in lib.dgm_last_error(), (kw, lib.dgm_last_error())
    for kw in (dict(m=0), dict(n=0)):
        assert lib.dgm_mxfp4_gemm_nt(ctypes.byref(_lib.Mxfp4GemmArgs(**{**gemm, **kw})), None) == 0
    assert lib.dgm_mxfp4_gemm_nt(None, None) == -1
    linear = dict(x=p, w=p, y=p, d_y=p, d_x=p, d_w=p, x_columns=p, x_column_scales=p, w_columns=p, w_column_scales=p, workspace=p,
                  workspace_bytes=1 << 30, m=4, n=8, k=64, x_stride=64, w_stride=64, d_y_stride=8)
    for fn, cases in ((lib.dgm_mxfp4_linear, ((dict(w=None), b"null pointer"), (dict(y=None), b"null pointer"), (dict(x_columns=None), b"their scales"))),
                      (lib.dgm_mxfp4_linear_backward, ((dict(d_y=None), b"null pointer"), (dict(w_columns=None, w_column_scales=None), b"forward pass"),
                                                       (dict(x_columns=None, x_column_scales=None), b"forward pass"), (dict(m=0), b"no tokens")))):
        for kw, what in cases + ((dict(x_dtype=3), b"dtypes"), (dict(w_dtype=-1), b"dtypes"), (dict(n=0), b"feature"), (dict(k=1 << 24), b"below 2^24"),
                                 (dict(workspace=None), b"workspace"), (dict(workspace=p + 8), b"workspace"), (dict(workspace_bytes=64), b"workspace")):
            st = fn(ctypes.byref(_lib.Mxfp4LinearArgs(**{**linear, **kw})), None)
            assert st == -1 and what in lib.dgm_last_error(), (kw, lib.dgm_last_error())
        assert fn(None, None) == -1
