"""The router's balance loss, per-expert counts and the gradient of its logits, on the GPU.

No counterpart in the reference, whose frontend stops at the top-k: this is what training the router, or
watching its balance in service, needs of the same logits and indices (``FusedSymmBuffer.logits`` and
``topk_idx`` as the frontend leaves them)."""
import ctypes
import functools

import torch

from . import _lib

MAX_EXPERTS = 1024
SCORES = {"softmax": 0, "sigmoid": 1}


def _rows(t):
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def _check(logits, topk_idx, cu_seqlens, score, z_coef):
    if logits.dim() != 2 or logits.dtype not in _lib.SRC_DTYPES:
        raise TypeError(f"logits must be bf16, fp16 or fp32 [tokens, experts], got {logits.dtype} {tuple(logits.shape)}")
    T, E = logits.shape
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"experts {E}: 1 to {MAX_EXPERTS}")
    if topk_idx.dim() != 2 or topk_idx.dtype not in (torch.int64, torch.int32) or topk_idx.size(0) != T:
        raise TypeError(f"topk_idx must be int64 or int32 [{T}, topk], got {topk_idx.dtype} {tuple(topk_idx.shape)}")
    if not 1 <= topk_idx.size(1) <= E or T * topk_idx.size(1) >= 1 << 31:
        raise ValueError(f"topk {topk_idx.size(1)}: 1 to {E}, tokens x topk below 2^31")
    if cu_seqlens is not None and (cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1
                                   or not 2 <= cu_seqlens.size(0) <= 1 << 21):
        raise TypeError(f"cu_seqlens must be int32 [sequences + 1], got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)} (below 2^21 sequences)")
    if score not in SCORES:
        raise ValueError(f"score {score!r}: one of {sorted(SCORES)}")
    if score == "sigmoid" and z_coef:
        raise ValueError("z_coef belongs to score='softmax'")
    _lib.no_tangents(logits)
    _lib.require_one_device(logits, topk_idx, cu_seqlens)


def _readable(logits, topk_idx, cu_seqlens):
    """The inputs as the kernels read them."""
    return _rows(logits), _rows(topk_idx), None if cu_seqlens is None else cu_seqlens.contiguous()


def _args(logits, topk_idx, cu_seqlens, balance_coef, z_coef, score, counts, stats):
    """DgmBalanceArgs of a call's inputs (logits and topk_idx as rows), counts and statistics."""
    T, E = logits.shape
    at = stats.data_ptr()                 # (per sequence 4 int32, then the totals)
    seqs = stats.size(0) // 4 - 1
    args = _lib.BalanceArgs(logits=logits.data_ptr(), topk_idx=topk_idx.data_ptr(), counts=counts.data_ptr(), seq_stats=at,
                            totals=at + 16 * seqs, tokens=T, logits_stride=logits.stride(0), idx_stride=topk_idx.stride(0),
                            experts=E, topk=topk_idx.size(1), seqs=seqs, dtype=_lib.SRC_DTYPES[logits.dtype],
                            idx_i64=int(topk_idx.dtype == torch.int64), score=SCORES[score],
                            balance_coef=float(balance_coef), z_coef=float(z_coef))
    if cu_seqlens is not None:
        args.cu_seqlens = cu_seqlens.data_ptr()
    return args


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(T, seqs, E):
    return _lib.load().dgm_router_balance_workspace_bytes(T, seqs, E)


def _forward(logits, topk_idx, cu_seqlens, balance_coef, z_coef, score):
    """The launches, after the checks: (loss, counts, stats, args, read). args: the launch's DgmBalanceArgs; read: the
    tensors whose memory it names."""
    dev = logits.device
    logits, topk_idx, cu_seqlens = _readable(logits, topk_idx, cu_seqlens)
    T, E = logits.shape
    seqs = 1 if cu_seqlens is None else cu_seqlens.size(0) - 1
    loss = torch.empty((), dtype=torch.float32, device=dev)
    counts = torch.empty((E,) if cu_seqlens is None else (seqs, E), dtype=torch.int32, device=dev)
    stats = torch.empty(4 * seqs + 4, dtype=torch.int32, device=dev)
    args = _args(logits, topk_idx, cu_seqlens, balance_coef, z_coef, score, counts, stats)
    args.loss = loss.data_ptr()
    need = _workspace_bytes(T, seqs, E)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _lib.check(_lib.load().dgm_router_balance_loss(ctypes.byref(args), _lib.stream()))
    return loss, counts, stats, args, (logits, topk_idx, cu_seqlens)


def _backward(d_loss, logits, args):
    """The launch of the backward pass, after the checks; args: DgmBalanceArgs of the forward call's inputs and results."""
    d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    args.d_loss, args.d_logits, args.d_logits_stride = d_loss.data_ptr(), d_logits.data_ptr(), logits.size(1)
    _lib.check(_lib.load().dgm_router_balance_loss_backward(ctypes.byref(args), _lib.stream()))
    return d_logits


def _check_backward(d_loss, logits, topk_idx, counts, stats, cu_seqlens, score, z_coef):
    _check(logits, topk_idx, cu_seqlens, score, z_coef)
    seqs = 1 if cu_seqlens is None else cu_seqlens.size(0) - 1
    E = logits.size(1)
    if (d_loss.dtype != torch.float32 or d_loss.numel() != 1 or counts.dtype != torch.int32 or counts.numel() != seqs * E
            or stats.dtype != torch.int32 or stats.numel() != 4 * seqs + 4 or not counts.is_contiguous()
            or not stats.is_contiguous()):
        raise TypeError("d_loss fp32 scalar, counts and stats of router_balance_loss_forward expected")
    _lib.no_tangents(d_loss)
    _lib.require_one_device(logits, d_loss, counts, stats)


def _places(tensors):
    return [None if t is None else (t.data_ptr(), t.stride()) for t in tensors]


class _RouterBalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk_idx, cu_seqlens, balance_coef, z_coef, score):
        loss, counts, stats, args, read = _forward(logits, topk_idx, cu_seqlens, balance_coef, z_coef, score)
        saved = logits, topk_idx, cu_seqlens, counts, stats
        ctx.save_for_backward(*saved)
        ctx.options, ctx.rows = (balance_coef, z_coef, score), (logits.dtype, logits.shape)
        # (the launch's arguments, those copies that the kernels read for inputs, and where the saved tensors were)
        ctx.args, ctx.copies, ctx.places = args, [None if u is t else u for t, u in zip(saved, read)], _places(saved)
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    def backward(ctx, d_loss, _):
        _lib.no_second_derivative()
        saved = ctx.saved_tensors
        logits, args = saved[0], ctx.args
        if _places(saved) != ctx.places:
            # Other memory since the forward pass, of saved-tensor hooks, which may bring anything back: checked as
            # arguments are, the kernel reads it by address.
            _, topk_idx, cu_seqlens, counts, stats = saved
            if (logits.dtype, logits.shape) != ctx.rows:
                raise TypeError(f"saved logits came back as {logits.dtype} {tuple(logits.shape)}")
            counts, stats = counts.contiguous(), stats.contiguous()
            _check_backward(d_loss, logits, topk_idx, counts, stats, cu_seqlens, ctx.options[2], ctx.options[1])
            held = _readable(logits, topk_idx, cu_seqlens)
            args = _args(*held, *ctx.options, counts, stats)
        _lib.no_tangents(d_loss, logits)
        return _backward(d_loss, logits, args), None, None, None, None, None


def router_balance_loss(logits, topk_idx, cu_seqlens=None, balance_coef=1.0, z_coef=0.0, score="softmax"):
    """The auxiliary loss that keeps experts evenly used, and their counts:

        loss = balance_coef * mean over sequences( sum_e f_e P_e ) + z_coef * mean over tokens( logsumexp^2 )

    f_e = experts * (slots of expert e) / (slots) and P_e = the mean of p_e over the sequence's routed
    tokens, p = softmax(logits) or, with ``score="sigmoid"``, sigmoid(logits) / their sum (then no z_coef).
    logits: bf16, fp16 or fp32 [tokens, experts <= 1024]; topk_idx: int64 or int32 [tokens, topk], ids
    outside [0, experts) are no slot (-1: unrouted), and a token without a slot adds nothing; cu_seqlens
    (int32 [sequences + 1], ascending): packed sequences, each with its own f and P, those without a routed
    token left out of the mean, tokens behind the last one ignored. An expert masked with -inf has p = 0.

    Returns ``(loss, counts)``: fp32 scalar and int32 [experts] (with cu_seqlens [sequences, experts]).
    Differentiable in logits through P and logsumexp (counts are constants); under graph capture use
    ``router_balance_loss_forward`` and ``router_balance_loss_backward``. Sums over tokens are taken in a
    fixed order. Work runs on the current stream of the tensors' device, which has to be the current one."""
    _check(logits, topk_idx, cu_seqlens, score, z_coef)
    if torch.is_grad_enabled() and logits.requires_grad:
        _lib.no_graph_under_capture()
        return _RouterBalanceLoss.apply(logits, topk_idx, cu_seqlens, float(balance_coef), float(z_coef), score)
    return _forward(logits, topk_idx, cu_seqlens, balance_coef, z_coef, score)[:2]


def router_balance_loss_forward(logits, topk_idx, cu_seqlens=None, balance_coef=1.0, z_coef=0.0, score="softmax"):
    """``router_balance_loss`` with what its explicit backward call needs: ``(loss, counts, stats)``. Records
    no autograd graph."""
    _check(logits, topk_idx, cu_seqlens, score, z_coef)
    return _forward(logits, topk_idx, cu_seqlens, balance_coef, z_coef, score)[:3]


def router_balance_loss_backward(d_loss, logits, topk_idx, counts, stats, cu_seqlens=None, balance_coef=1.0, z_coef=0.0,
                                 score="softmax"):
    """The logits' gradient (logits' type) from d_loss (fp32 scalar tensor), the forward call's inputs and the
    counts and stats of ``router_balance_loss_forward``; zeros for tokens that add nothing."""
    _check_backward(d_loss, logits, topk_idx, counts, stats, cu_seqlens, score, z_coef)
    held = _readable(logits, topk_idx, cu_seqlens)
    return _backward(d_loss, logits, _args(*held, balance_coef, z_coef, score, counts, stats))


__all__ = ["router_balance_loss", "router_balance_loss_forward", "router_balance_loss_backward"]
