"""router_balance_loss: what is refused before any GPU work (CPU)."""
import ctypes

import pytest
import torch

import hopper_megamoe_basedondeepgemm_amd as dgm
from hopper_megamoe_basedondeepgemm_amd import _lib


def idx(t, k, dtype=torch.int64):
    return torch.zeros((t, k), dtype=dtype)


def test_struct_size():
    a = ctypes.c_size_t(0)
    assert _lib.load().dgm_balance_struct_size(ctypes.byref(a)) == 0 and a.value == ctypes.sizeof(_lib.BalanceArgs)


@pytest.mark.parametrize("args, kw, err, what", [
    ((torch.zeros(4), idx(4, 2)), {}, TypeError, "logits must be"),
    ((torch.zeros(4, 8, dtype=torch.float64), idx(4, 2)), {}, TypeError, "logits must be"),
    ((torch.zeros(4, 1025), idx(4, 2)), {}, ValueError, "experts 1025"),
    ((torch.zeros(4, 0), idx(4, 2)), {}, ValueError, "experts 0"),
    ((torch.zeros(4, 8), idx(5, 2)), {}, TypeError, "topk_idx must be"),
    ((torch.zeros(4, 8), idx(4, 2, torch.int16)), {}, TypeError, "topk_idx must be"),
    ((torch.zeros(4, 8), idx(4, 9)), {}, ValueError, "topk 9"),
    ((torch.zeros(4, 8), idx(4, 0)), {}, ValueError, "topk 0"),
    ((torch.zeros(4, 8), idx(4, 2), torch.tensor([0, 4])), {}, TypeError, "cu_seqlens must be"),
    ((torch.zeros(4, 8), idx(4, 2), torch.tensor([0], dtype=torch.int32)), {}, TypeError, "cu_seqlens must be"),
    ((torch.zeros(4, 8), idx(4, 2), torch.zeros((1 << 21) + 1, dtype=torch.int32)), {}, TypeError, "cu_seqlens must be"),
    ((torch.zeros(4, 8), idx(4, 2)), dict(score="tanh"), ValueError, "score"),
    ((torch.zeros(4, 8), idx(4, 2)), dict(score="sigmoid", z_coef=0.1), ValueError, "z_coef"),
    ((torch.zeros(4, 8), idx(4, 2)), {}, RuntimeError, "GPU"),
])
def test_refusals(args, kw, err, what):
    with pytest.raises(err, match=what):
        dgm.router_balance_loss(*args, **kw)


def test_c_entry_refusals():
    lib, p = _lib.load(), 4096          # (never dereferenced: refused first)
    base = dict(logits=p, topk_idx=p, loss=p, counts=p, seq_stats=p, totals=p, tokens=1000, logits_stride=8, idx_stride=2,
                experts=8, topk=2, seqs=1, dtype=2, idx_i64=1)
    for kw, what in ((dict(dtype=3), b"dtype"), (dict(experts=0), b"experts"), (dict(experts=1025), b"experts"),
                     (dict(topk=9), b"topk"), (dict(topk=0), b"topk"), (dict(tokens=-1), b"tokens"),
                     (dict(tokens=1 << 30), b"tokens"), (dict(seqs=0), b"seqs"), (dict(seqs=2), b"seqs"), (dict(seqs=1 << 21, cu_seqlens=p), b"seqs"),
                     (dict(score=2), b"score"), (dict(score=1, z_coef=0.5), b"score"), (dict(counts=None), b"null"),
                     (dict(logits=None), b"null"), (dict(loss=None), b"null loss"), ({}, b"workspace"),
                     (dict(workspace=p, workspace_bytes=lib.dgm_router_balance_workspace_bytes(1000, 1, 8) - 1), b"workspace"),
                     (dict(workspace=p + 8, workspace_bytes=1 << 30), b"workspace")):
        st = lib.dgm_router_balance_loss(ctypes.byref(_lib.BalanceArgs(**{**base, **kw})), None)
        assert st == -1 and what in lib.dgm_last_error(), (kw, lib.dgm_last_error())
    st = lib.dgm_router_balance_loss_backward(ctypes.byref(_lib.BalanceArgs(**base)), None)
    assert st == -1 and b"null" in lib.dgm_last_error()
    assert lib.dgm_router_balance_loss_backward(ctypes.byref(_lib.BalanceArgs(**{**base, "tokens": 0})), None) == 0
    assert lib.dgm_router_balance_loss(None, None) == -1 and lib.dgm_router_balance_loss_backward(None, None) == -1
    assert lib.dgm_router_balance_workspace_bytes(256, 1, 8) == 0 and lib.dgm_router_balance_workspace_bytes(257, 1, 8) > 0
