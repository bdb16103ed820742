"""rms_norm_residual: what is refused before any GPU work (CPU)."""
import ctypes

import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm
from hopper_megamoe_basedondeepgemm_amd import _lib


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_struct_sizes():
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert _lib.load().dgm_norm_struct_sizes(ctypes.byref(a), ctypes.byref(b)) == 0
    assert (a.value, b.value) == (ctypes.sizeof(_lib.NormArgs), ctypes.sizeof(_lib.NormGradArgs))


@pytest.mark.parametrize("kw, err, what", [
    (dict(x=bf(4)), TypeError, "bf16, fp16 or fp32"),
    (dict(x=torch.zeros(4, 8, dtype=torch.int8)), TypeError, "bf16, fp16 or fp32"),
    (dict(x=bf(1, 16385)), ValueError, "hidden 16385"),
    (dict(x=bf(4, 0)), ValueError, "hidden 0"),
    (dict(x=bf(1, 1).expand(1 << 22, 1)), ValueError, "tokens 4194304"),
    (dict(x=bf(4, 8), residual=bf(4, 9)), TypeError, "rows of"),
    (dict(x=bf(4, 8), residual=torch.zeros(4, 8)), TypeError, "rows of"),
    (dict(x=bf(4, 8), pre_weight=bf(9)), TypeError, "norm weights"),
    (dict(x=bf(4, 8), pre_weight=torch.zeros(8, dtype=torch.float16)), TypeError, "norm weights"),
    (dict(x=bf(4, 8), pre_weight=bf(8), post_weight=torch.zeros(8)), TypeError, "norm weights"),
    (dict(x=bf(4, 8), gate=torch.zeros(8)), TypeError, "gate of"),
    (dict(x=bf(4, 8), gate=bf(4)), ValueError, "gate of shape"),
    (dict(x=bf(4, 8), gate=bf(1, 8)), ValueError, "gate of shape"),
    (dict(x=bf(4, 8), pre_weight=bf(8), quant="fp8"), ValueError, "quant"),
    (dict(x=bf(4, 8), quant="int8"), ValueError, "int8 rows"),
    (dict(x=torch.zeros(4, 8), pre_weight=torch.zeros(8), quant="int8"), ValueError, "int8 rows"),
    (dict(x=bf(4, 8), out=bf(4, 8)), ValueError, "pre_weight only"),
    (dict(x=bf(4, 8), residual_out=bf(8, 4).t()), ValueError, "contiguous"),
    (dict(x=bf(4, 8), residual_out=bf(1, 8).expand(4, 8)), ValueError, "overlap"),
    (dict(x=bf(4, 8)), RuntimeError, "GPU"),
])
def test_refusals(kw, err, what):
    with pytest.raises(err, match=what):
        dgm.rms_norm_residual(**kw)


def test_backward_refusals():
    x, w = bf(4, 8), bf(8)
    rstd = torch.zeros(4)
    with pytest.raises(TypeError, match="gradient rows"):
        dgm.rms_norm_residual_backward(None, bf(4, 9), x, None, None, rstd, pre_weight=w)
    with pytest.raises(ValueError, match="without a pre_weight"):
        dgm.rms_norm_residual_backward(None, bf(4, 8), x, None, None, None)
    with pytest.raises(ValueError, match="rstd rows"):
        dgm.rms_norm_residual_backward(None, bf(4, 8), x, None, None, None, pre_weight=w)
    with pytest.raises(RuntimeError, match="GPU"):
        dgm.rms_norm_residual_backward(None, bf(4, 8), x, None, None, rstd, pre_weight=w)


def test_c_entry_refusals():
    lib, p = _lib.load(), 4096          # (never dereferenced: refused first)
    base = dict(x=p, h=p, pre_weight=p, rows=4, hidden=64, x_stride=64, h_stride=64, residual_scale=1.0, eps=1e-6)
    for kw, what in ((dict(dtype=3), b"dtype"), (dict(hidden=0), b"hidden"), (dict(hidden=16385), b"hidden"),
                     (dict(rows=-1), b"rows"), (dict(rows=1 << 22), b"rows"), (dict(gate_mode=4), b"gate_mode"), (dict(gate_mode=1), b"gate and gate_mode"),
                     (dict(x=None), b"null x"), (dict(eps=-1.0), b"eps"), (dict(q=p), b"int8 rows"),
                     (dict(q=p, q_sf=p, dtype=2), b"int8 rows")):
        st = lib.dgm_rms_norm_residual(ctypes.byref(_lib.NormArgs(**{**base, **kw})), None)
        assert st == -1 and what in lib.dgm_last_error(), (kw, lib.dgm_last_error())
    assert lib.dgm_rms_norm_residual(ctypes.byref(_lib.NormArgs(**{**base, "rows": 0})), None) == 0
    assert lib.dgm_rms_norm_residual(None, None) == -1

    def grad(fwd, **kw):
        a = _lib.NormGradArgs(forward=_lib.NormArgs(**{**base, **fwd}), **kw)
        return lib.dgm_rms_norm_residual_backward(ctypes.byref(a), None), lib.dgm_last_error()
    groups = lib.dgm_rms_norm_residual_groups(4, 64)
    for fwd, kw, what in (({}, dict(d_h=p), b"rstd_pre"), (dict(post_weight=p), {}, b"rstd_post"),
                          (dict(rstd_pre=p), dict(d_h=p, d_pre_weight=p), b"workspace"),
                          (dict(rstd_pre=p), dict(d_h=p, d_pre_weight=p, workspace=p,
                                                  workspace_bytes=groups * 64 * 12 - 1), b"workspace"),
                          ({}, dict(d_residual=p), b"d_residual"), ({}, dict(d_gate=p), b"d_gate"),
                          ({}, dict(d_post_weight=p), b"d_post_weight")):
        st, msg = grad(fwd, **kw)
        assert st == -1 and what in msg, (fwd, kw, msg)


def test_c_backward_without_rows():
    """No rows: a channel gate is read all the same, so a null one is refused."""
    lib, p = _lib.load(), 4096          # (never dereferenced: refused first)
    for hidden in (64, 9000):
        fwd = _lib.NormArgs(rows=0, hidden=hidden, gate_mode=1, residual_scale=1.0, eps=1e-6)
        a = _lib.NormGradArgs(forward=fwd, d_gate=p, workspace=p, workspace_bytes=hidden * 12)
        assert lib.dgm_rms_norm_residual_backward(ctypes.byref(a), None) == -1
        assert b"gate and gate_mode" in lib.dgm_last_error()
