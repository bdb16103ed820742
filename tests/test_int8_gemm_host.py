"""int8_gemm_nt: what is refused before any GPU work (CPU)."""
import ctypes

import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm
from hopper_megamoe_basedondeepgemm_amd import _lib


def rows(m, k):
    return torch.zeros((m, k), dtype=torch.int8), torch.zeros(m)


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_struct_size():
    a = ctypes.c_size_t(0)
    assert _lib.load().dgm_int8_gemm_struct_size(ctypes.byref(a)) == 0 and a.value == ctypes.sizeof(_lib.Int8GemmArgs)


@pytest.mark.parametrize("a, b, d, kw, err, what", [
    ((bf(4, 32), torch.zeros(4)), rows(8, 32), bf(4, 8), {}, TypeError, "a: int8"),
    (rows(4, 32), (rows(8, 32)[0], torch.zeros(7)), bf(4, 8), {}, TypeError, "b: fp32 scales"),
    ((rows(4, 32)[0], bf(4)), rows(8, 32), bf(4, 8), {}, TypeError, "a: fp32 scales"),
    ((rows(4, 32)[0], torch.zeros(4, 0)), rows(8, 32), bf(4, 8), {}, TypeError, "a: fp32 scales"),
    (rows(4, 32), rows(8, 48), bf(4, 8), {}, ValueError, "k of a"),
    (rows(4, 0), rows(8, 0), bf(4, 8), {}, ValueError, "k of a"),
    (rows(1, 131072), rows(1, 131072), bf(1, 1), {}, ValueError, "k of a"),
    (rows(4, 32), rows(8, 32), bf(4, 9), {}, TypeError, "d: bf16"),
    (rows(4, 32), rows(8, 32), torch.zeros((4, 8), dtype=torch.float64), {}, TypeError, "d: bf16"),
    (rows(4, 32), rows(8, 32), bf(8, 4).t(), {}, ValueError, "d: rows"),
    (rows(4, 32), rows(8, 32), bf(1, 8).expand(4, 8), {}, ValueError, "d: rows"),
    (rows(4, 32), rows(8, 32), bf(4, 8), dict(c=torch.zeros(4, 8)), TypeError, "c: "),
    (rows(4, 32), rows(8, 32), bf(4, 8), dict(c=bf(4)), TypeError, "c: "),
    (rows(4, 32), rows(8, 32), bf(4, 8), dict(activation="gelu"), ValueError, "activation"),
    (rows(4, 32), rows(7, 32), bf(4, 3), dict(activation="swiglu"), ValueError, "swiglu"),
    (rows(4, 32), rows(8, 32), bf(4, 4), dict(activation="swiglu", c=bf(4, 4)), ValueError, "swiglu"),
    (rows(4, 32), rows(8, 32), bf(4, 4), dict(activation="swiglu", activation_clamp=-1.0), ValueError, "activation_clamp"),
    (rows(4, 32), rows(8, 32), bf(4, 4), dict(activation="swiglu", activation_clamp=float("nan")), ValueError, "activation_clamp"),
    (rows(4, 32), rows(8, 32), bf(4, 8), {}, RuntimeError, "GPU"),
])
def test_refusals(a, b, d, kw, err, what):
    with pytest.raises(err, match=what):
        dgm.int8_gemm_nt(a, b, d, **kw)


@pytest.mark.parametrize("leaf", ["sfa", "sfb", "c", "d"])
def test_no_gradient_is_dropped(leaf):
    """A product, or a block, over leaves that ask for a gradient is refused, their scales among them."""
    a, b, d, c = rows(4, 32), rows(8, 32), torch.zeros(4, 8), torch.zeros(4, 8)
    {"sfa": a[1], "sfb": b[1], "c": c, "d": d}[leaf].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        dgm.int8_gemm_nt(a, b, d, c=c)
    with pytest.raises(RuntimeError, match="GPU"), torch.no_grad():
        dgm.int8_gemm_nt(a, b, d, c=c)
    if leaf == "sfb":
        with pytest.raises(RuntimeError, match="no gradient"):
            dgm.mega_moe_block(bf(4, 32), bf(32), bf(2, 32), None, None, None, shared_expert=(b, a))


def test_c_entry_refusals():
    lib, p = _lib.load(), 4096          # (never dereferenced: refused first)
    base = dict(a=p, sfa=p, b=p, sfb=p, d=p, m=4, n=8, k=32, a_stride=32, b_stride=32, d_stride=8, sfa_stride=1, sfb_stride=1)
    for kw, what in ((dict(dtype=3), b"dtype"), (dict(k=0), b"k 1 to"), (dict(k=131072), b"k 1 to"), (dict(m=-1), b"m below"),
                     (dict(m=1 << 20), b"m below"), (dict(n=1 << 24), b"n below"), (dict(swiglu=1, c=p), b"SwiGLU"),
                     (dict(swiglu=1, n=7), b"SwiGLU"), (dict(a_stride=-1), b"strides"), (dict(d=None), b"null pointer")):
        st = lib.dgm_int8_gemm_nt(ctypes.byref(_lib.Int8GemmArgs(**{**base, **kw})), None)
        assert st == -1 and what in lib.dgm_last_error(), (kw, lib.dgm_last_error())
    for kw in (dict(m=0), dict(n=0)):
        assert lib.dgm_int8_gemm_nt(ctypes.byref(_lib.Int8GemmArgs(**{**base, **kw})), None) == 0
    assert lib.dgm_int8_gemm_nt(None, None) == -1
