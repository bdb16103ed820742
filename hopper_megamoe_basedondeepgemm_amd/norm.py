"""Norms around a block with its gate and scaled residual add, on the GPU, and their gradients.

No counterpart in the reference, whose layer starts at the router: these are the row passes that a
decoder block needs before ``fable_router_quant_topk_frontend`` and behind the layer's combine."""
import ctypes
import functools

import torch

from . import _lib

MAX_HIDDEN, MAX_TOKENS = 16384, 1 << 22
GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_FULL = 0, 1, 2, 3


def _rows(t):
    """t as the kernels read it: rows of contiguous elements (any row stride)."""
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def _new_like(t):
    """An uninitialised contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _gate_mode(gate, T, H):
    shape = tuple(gate.shape)
    if shape == (H,):
        return GATE_CHANNEL
    if shape == (T, 1):
        return GATE_TOKEN
    if shape == (T, H):
        return GATE_FULL
    raise ValueError(f"gate of shape {shape}: [hidden], [tokens, 1] or [tokens, hidden]")


def _check(x, residual, post_weight, pre_weight, gate, quant=None, residual_out=None, out=None):
    if x.dim() != 2 or x.dtype not in _lib.SRC_DTYPES:
        raise TypeError(f"x must be bf16, fp16 or fp32 [tokens, hidden], got {x.dtype} {tuple(x.shape)}")
    T, H = x.shape
    if not 1 <= H <= MAX_HIDDEN:
        raise ValueError(f"hidden {H}: 1 to {MAX_HIDDEN}")
    if T >= MAX_TOKENS:
        raise ValueError(f"tokens {T}: below {MAX_TOKENS}")
    for t in (residual, residual_out, out):
        if t is not None and (t.dtype != x.dtype or t.shape != x.shape):
            raise TypeError(f"rows of {x.dtype} {tuple(x.shape)} expected, got {t.dtype} {tuple(t.shape)}")
    wdt = None
    for w in (post_weight, pre_weight):
        if w is not None:
            if w.dim() != 1 or w.size(0) != H or w.dtype not in (x.dtype, torch.float32) or wdt not in (None, w.dtype):
                raise TypeError(f"norm weights must be [hidden] of {x.dtype} or fp32, both of one type; got "
                                f"{w.dtype} {tuple(w.shape)}")
            wdt = w.dtype
    if gate is not None and gate.dtype != x.dtype:
        raise TypeError(f"gate of {x.dtype} expected, got {gate.dtype}")
    if quant not in (None, "int8"):
        raise ValueError(f"quant {quant!r}: None or 'int8'")
    if quant and (x.dtype != torch.bfloat16 or pre_weight is None):
        raise ValueError("int8 rows are cast from bf16 rows and need a pre_weight")
    for t in (residual_out, out):
        if t is not None and t.numel() and t.stride(1) != 1 and H > 1:
            raise ValueError("output rows must be contiguous")
        if t is not None and T > 1 and t.stride(0) < H:
            raise ValueError("output rows overlap")
    if out is not None and pre_weight is None:
        raise ValueError("out is written with a pre_weight only")
    if gate is not None:
        _gate_mode(gate, T, H)


def _same_rows(a, b):
    return a.data_ptr() == b.data_ptr() and a.stride(0) == b.stride(0)


def _span(t):
    return t.data_ptr(), t.data_ptr() + ((t.size(0) - 1) * t.stride(0) + t.size(1)) * t.element_size()


def _check_outputs(outs, ins):
    """An output may be an input's own rows (each row is read before it is written), nothing else that overlaps."""
    for i, o in enumerate(outs):
        lo, hi = _span(o)
        for t in outs[:i]:
            a, z = _span(t)
            if lo < z and a < hi:
                raise ValueError("the outputs overlap")
        for t in ins:
            a, z = _span(t if t.dim() == 2 else t[None])
            if lo < z and a < hi and not (t.dim() == 2 and t.shape == o.shape and _same_rows(o, t)):
                raise ValueError("an output overlaps an input other than as the same rows")


def _forward_args(x, residual, post_weight, pre_weight, gate, gate_sigmoid, residual_scale, eps, mode, rstd_post, rstd_pre):
    """DgmNormArgs of a call's inputs. (The fields of absent parts stay at their zero: each one set costs time on
    a call that the GPU finishes in 3 us.)"""
    T, H = x.shape
    w = post_weight if post_weight is not None else pre_weight
    args = _lib.NormArgs(x=x.data_ptr(), rows=T, x_stride=x.stride(0), hidden=H, dtype=_lib.SRC_DTYPES[x.dtype],
                         residual_scale=float(residual_scale), eps=float(eps))
    if residual is not None:
        args.residual, args.residual_stride = residual.data_ptr(), residual.stride(0)
    if post_weight is not None:
        args.post_weight, args.rstd_post = post_weight.data_ptr(), rstd_post
    if pre_weight is not None:
        args.pre_weight, args.rstd_pre = pre_weight.data_ptr(), rstd_pre
    if w is not None and w.dtype == torch.float32:
        args.weights_f32 = 1
    if gate is not None:
        args.gate, args.gate_mode, args.gate_sigmoid = gate.data_ptr(), mode, int(bool(gate_sigmoid))
        if mode != GATE_CHANNEL:
            args.gate_stride = gate.stride(0)
    return args


def _readable(x, residual, post_weight, pre_weight, gate):
    """The inputs as the kernels read them, and the gate's mode."""
    x = _rows(x)
    if residual is not None:
        residual = _rows(residual)
    if post_weight is not None and post_weight.stride(0) != 1:
        post_weight = post_weight.contiguous()
    if pre_weight is not None and pre_weight.stride(0) != 1:
        pre_weight = pre_weight.contiguous()
    mode = GATE_NONE
    if gate is not None:
        mode = _gate_mode(gate, x.size(0), x.size(1))
        if mode == GATE_FULL:
            gate = _rows(gate)
        elif mode == GATE_CHANNEL:
            gate = gate.contiguous()
    return x, residual, post_weight, pre_weight, gate, mode


def _forward(x, residual, post_weight, pre_weight, gate, gate_sigmoid, residual_scale, eps, quant, residual_out, out, keep):
    """The launch, after the checks: (residual rows, h, q, sf, rstd, args, read). ``keep``: rstd fp32 [norms,
    tokens] for the backward pass; args: the launch's DgmNormArgs; read: the tensors whose memory it names."""
    T = x.size(0)
    read = _readable(x, residual, post_weight, pre_weight, gate)
    x_, residual_, post_, pre_, gate_, mode = read
    same = residual is None and post_weight is None and gate is None and residual_scale == 1.0 and residual_out is None
    r_out = None if same else residual_out if residual_out is not None else _new_like(x)
    h = None if pre_weight is None else out if out is not None else _new_like(x)
    q = sf = rstd = None
    at = 0
    if keep:
        rstd = torch.empty(((post_weight is not None) + (pre_weight is not None), T), dtype=torch.float32, device=x.device)
        at = rstd.data_ptr()
    args = _forward_args(x_, residual_, post_, pre_, gate_, gate_sigmoid, residual_scale, eps, mode, at,
                         at + 4 * T if at and post_weight is not None else at)
    if r_out is not None:
        args.residual_out, args.residual_out_stride = r_out.data_ptr(), r_out.stride(0)
    if h is not None:
        args.h, args.h_stride = h.data_ptr(), h.stride(0)
    if quant:
        q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        sf = torch.empty((T,), dtype=torch.float32, device=x.device)
        args.q, args.q_sf = q.data_ptr(), sf.data_ptr()
    if (residual_out is not None or out is not None) and T > 0:
        _check_outputs([t for t in (residual_out, out) if t is not None], [t for t in read[:5] if t is not None])
    if T > 0 and not (same and h is None):
        _lib.check(_lib.load().dgm_rms_norm_residual(ctypes.byref(args), _lib.stream()))
        if residual_out is not None or out is not None:
            _lib.written(*(t for t in (residual_out, out) if t is not None))
    return x if same else r_out, h, q, sf, rstd, args, read


@functools.lru_cache(maxsize=1024)
def _groups(T, H):
    return _lib.load().dgm_rms_norm_residual_groups(T, H)


def _backward(d_r, d_h, x, residual, post_weight, pre_weight, gate, forward, needs):
    """The launches of the backward pass, after the checks; forward: DgmNormArgs over the forward call's inputs
    and rstd rows."""
    T, H = x.shape
    args = _lib.NormGradArgs(forward)
    if d_r is not None:
        d_r = _rows(d_r)
        args.d_residual_out, args.d_residual_out_stride = d_r.data_ptr(), d_r.stride(0)
    if d_h is not None:
        d_h = _rows(d_h)
        args.d_h, args.d_h_stride = d_h.data_ptr(), d_h.stride(0)
    d_x = d_residual = d_post = d_pre = d_gate = None
    columns = False                       # (a gradient that is a sum over rows)
    if needs[0]:
        d_x = _new_like(x)
        args.d_x, args.d_x_stride = d_x.data_ptr(), H
    if needs[1] and residual is not None:
        d_residual = _new_like(x)
        args.d_residual, args.d_residual_stride = d_residual.data_ptr(), H
    if needs[2] and post_weight is not None:
        d_post = _new_like(post_weight)
        args.d_post_weight = d_post.data_ptr()
        columns = True
    if needs[3] and pre_weight is not None:
        d_pre = _new_like(pre_weight)
        args.d_pre_weight = d_pre.data_ptr()
        columns = True
    if needs[4] and gate is not None:
        d_gate = _new_like(gate)
        args.d_gate = d_gate.data_ptr()
        if forward.gate_mode == GATE_CHANNEL:
            columns = True
        else:
            args.d_gate_stride = d_gate.size(1)
    if columns:
        ws = torch.empty(3 * _groups(T, H) * H, dtype=torch.float32, device=x.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.nbytes
    _lib.check(_lib.load().dgm_rms_norm_residual_backward(ctypes.byref(args), _lib.stream()))
    return d_x, d_residual, d_post, d_pre, d_gate


def _check_backward(d_r, d_h, x, residual, post_weight, pre_weight, gate, rstd_post, rstd_pre):
    _check(x, residual, post_weight, pre_weight, gate)
    for d in (d_r, d_h):
        if d is not None and (d.dtype != x.dtype or d.shape != x.shape):
            raise TypeError(f"gradient rows of {x.dtype} {tuple(x.shape)} expected, got {d.dtype} {tuple(d.shape)}")
    if d_h is not None and pre_weight is None:
        raise ValueError("d_h without a pre_weight")
    for w, rstd in ((post_weight, rstd_post), (pre_weight, rstd_pre)):
        if w is not None and (rstd is None or rstd.dtype != torch.float32 or tuple(rstd.shape) != (x.size(0),)
                              or not rstd.is_contiguous()):
            raise ValueError("rstd rows of rms_norm_residual_forward (fp32 [tokens]) expected")
    _lib.require_one_device(x, d_r, d_h, residual, post_weight, pre_weight, gate, rstd_post, rstd_pre)


def _places(tensors):
    return [None if t is None else (t.data_ptr(), t.stride()) for t in tensors]


class _RmsNormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, post_weight, pre_weight, gate, gate_sigmoid, residual_scale, eps):
        r, h, _, _, rstd, args, read = _forward(x, residual, post_weight, pre_weight, gate, gate_sigmoid, residual_scale, eps,
                                                None, None, None, True)
        saved = x, residual, post_weight, pre_weight, gate, rstd
        ctx.save_for_backward(*saved)
        ctx.options = gate_sigmoid, residual_scale, eps
        # (the launch's arguments, those copies that the kernels read for inputs, and where the saved tensors were)
        ctx.args, ctx.copies, ctx.places = args, [None if u is t else u for t, u in zip(saved, read[:5])], _places(saved)
        ctx.set_materialize_grads(False)
        return (None if r is x else r), h

    @staticmethod
    def backward(ctx, d_r, d_h):
        _lib.no_second_derivative()
        saved = ctx.saved_tensors
        _lib.no_tangents(d_r, d_h, *saved)
        args = ctx.args
        if _places(saved) != ctx.places:
            # Other memory since the forward pass: storage replaced, or tensors that saved-tensor hooks brought
            # back (offloading, recomputation), the rstd rows among them and in strides of their own. What a hook
            # returns is checked as an argument is: the kernels read it by address.
            rstd = saved[5].contiguous()
            post, pre = saved[2] is not None, saved[3] is not None
            if rstd.dim() != 2 or rstd.size(0) != post + pre:
                raise ValueError(f"saved rstd rows came back as {tuple(rstd.shape)}")
            _check_backward(d_r, d_h, *saved[:5], rstd[0] if post else None, rstd[-1] if pre else None)
            read = _readable(*saved[:5])
            at = rstd.data_ptr()
            args = _forward_args(*read[:5], *ctx.options, read[5], at, at + 4 * rstd.size(1) if post else at)
        return (*_backward(d_r, d_h, *saved[:5], args, ctx.needs_input_grad), None, None, None)


def rms_norm_residual(x, residual=None, post_weight=None, pre_weight=None, gate=None, gate_sigmoid=False,
                      residual_scale=1.0, eps=1e-6, quant=None, residual_out=None, out=None):
    """The norm behind a block, its gate, the scaled residual add and the norm before the next block, in
    one pass over the rows:

        n = x / sqrt(mean(x^2) + eps) * post_weight       (n = x without post_weight)
        r = residual + residual_scale * a * n             (a = gate, or sigmoid(gate) with gate_sigmoid)
        h = r / sqrt(mean(r^2) + eps) * pre_weight

    x, residual: bf16, fp16 or fp32 [tokens < 2^22, hidden <= 16384], any row stride; norm weights [hidden] of
    that type or fp32; gate [hidden], [tokens, 1] or [tokens, hidden]. Every part but x may be absent.
    Arithmetic in fp32 (the squares of a row have to add up below 3.4e38); r enters the second norm
    unrounded. Returns ``(r, h)``, h None without pre_weight, r x itself where nothing changes it; with
    ``quant="int8"`` (bf16) ``(r, h, (q, sf))``: the int8 rows and scales [tokens] of the rounded h
    (bit for bit ``per_token_cast_to_int8(h)``), as ``int8_gemm_nt`` takes them. ``residual_out`` /
    ``out``: where r and h go; either may be x's or residual's own rows.

    Differentiable in x, residual, gate and the weights (not with quant, residual_out or out; under graph
    capture use ``rms_norm_residual_forward`` and ``rms_norm_residual_backward``). Work runs on the
    current stream of the tensors' device, which has to be the current one."""
    _check(x, residual, post_weight, pre_weight, gate, quant, residual_out, out)
    _lib.no_tangents(x, residual, post_weight, pre_weight, gate, residual_out, out)
    _lib.require_one_device(x, residual, post_weight, pre_weight, gate, residual_out, out)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)
                                    or (post_weight is not None and post_weight.requires_grad)
                                    or (pre_weight is not None and pre_weight.requires_grad)
                                    or (gate is not None and gate.requires_grad)
                                    or (residual_out is not None and residual_out.requires_grad)
                                    or (out is not None and out.requires_grad)):
        _lib.no_graph_under_capture()
        if quant or residual_out is not None or out is not None:
            raise ValueError("quant, residual_out and out have no gradient: call under torch.no_grad()")
        r, h = _RmsNormResidual.apply(x, residual, post_weight, pre_weight, gate, bool(gate_sigmoid),
                                      float(residual_scale), float(eps))
        return (x if r is None else r), h
    r, h, q, sf, _, _, _ = _forward(x, residual, post_weight, pre_weight, gate, gate_sigmoid, residual_scale, eps, quant,
                                    residual_out, out, False)
    return (r, h, (q, sf)) if quant else (r, h)


def rms_norm_residual_forward(x, residual=None, post_weight=None, pre_weight=None, gate=None, gate_sigmoid=False,
                              residual_scale=1.0, eps=1e-6):
    """``rms_norm_residual`` with what its explicit backward call needs: ``(r, h, rstd_post, rstd_pre)``
    (fp32 [tokens] each, None without that norm). Records no autograd graph."""
    _check(x, residual, post_weight, pre_weight, gate)
    _lib.no_tangents(x, residual, post_weight, pre_weight, gate)
    _lib.require_one_device(x, residual, post_weight, pre_weight, gate)
    r, h, _, _, rstd, _, _ = _forward(x, residual, post_weight, pre_weight, gate, gate_sigmoid, residual_scale, eps, None,
                                      None, None, True)
    return r, h, rstd[0] if post_weight is not None else None, rstd[-1] if pre_weight is not None else None


def rms_norm_residual_backward(d_r, d_h, x, residual, rstd_post, rstd_pre, post_weight=None, pre_weight=None, gate=None,
                               gate_sigmoid=False, residual_scale=1.0, eps=1e-6, needs=(True,) * 5):
    """Gradients of ``rms_norm_residual``: ``(d_x, d_residual, d_post_weight, d_pre_weight, d_gate)`` from
    d_r = dL/dr and d_h = dL/dh (either may be None: zero), the forward call's inputs and the rstd rows of
    ``rms_norm_residual_forward``; None for an absent input or one that ``needs`` leaves out. r is
    recomputed in fp32 from x and residual. Sums over tokens (the weights, a channel gate) are taken in
    fp32 in a fixed order."""
    _check_backward(d_r, d_h, x, residual, post_weight, pre_weight, gate, rstd_post, rstd_pre)
    _lib.no_tangents(d_r, d_h, x, residual, post_weight, pre_weight, gate)
    read = _readable(x, residual, post_weight, pre_weight, gate)
    forward = _forward_args(*read[:5], gate_sigmoid, residual_scale, eps, read[5],
                            rstd_post.data_ptr() if post_weight is not None else 0,
                            rstd_pre.data_ptr() if pre_weight is not None else 0)
    return _backward(d_r, d_h, x, residual, post_weight, pre_weight, gate, forward, needs)


__all__ = ["rms_norm_residual", "rms_norm_residual_forward", "rms_norm_residual_backward"]
