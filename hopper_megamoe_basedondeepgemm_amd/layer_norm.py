"""Scaled residual add and layer norm, on the GPU, and their gradients: what ``rms_norm_residual`` is for blocks whose
norm takes the mean off and has a bias. No counterpart in the reference, whose layer starts at the router."""
import ctypes
import functools

import torch

from . import _lib
from .mxfp4 import _new as _new_mxfp4, _quantize
from .norm import MAX_HIDDEN, MAX_TOKENS, _check_outputs, _new_like, _places, _rows


def _check(x, residual, weight, bias, quant=None, residual_out=None, out=None):
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
    for w in (weight, bias):
        if w is not None:
            if w.dim() != 1 or w.size(0) != H or w.dtype not in (x.dtype, torch.float32) or wdt not in (None, w.dtype):
                raise TypeError(f"weight and bias must be [hidden] of {x.dtype} or fp32, both of one type; got "
                                f"{w.dtype} {tuple(w.shape)}")
            wdt = w.dtype
    if quant not in (None, "mxfp4"):
        raise ValueError(f"quant {quant!r}: None or 'mxfp4'")
    if quant and x.dtype != torch.bfloat16:
        raise ValueError("MXFP4 rows are cast from bf16 rows")
    for t in (residual_out, out):
        if t is not None and t.numel() and t.stride(1) != 1 and H > 1:
            raise ValueError("output rows must be contiguous")
        if t is not None and T > 1 and t.stride(0) < H:
            raise ValueError("output rows overlap")


def _forward_args(x, residual, weight, bias, residual_scale, eps):
    """DgmLayerNormArgs of a call's inputs (its outputs at their zero)."""
    T, H = x.shape
    w = weight if weight is not None else bias
    r, r_stride = (0, 0) if residual is None else (residual.data_ptr(), residual.stride(0))
    return _lib.LayerNormArgs(x.data_ptr(), r, 0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
                              0, 0, 0, 0, 0, 0, T, x.stride(0), r_stride, 0, 0, H, _lib.SRC_DTYPES[x.dtype],
                              w is not None and w.dtype == torch.float32, residual_scale, eps)


def _readable(x, residual, weight, bias):
    """The inputs as the kernels read them."""
    x = _rows(x)
    if residual is not None:
        residual = _rows(residual)
    if weight is not None and weight.stride(0) != 1:
        weight = weight.contiguous()
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    return x, residual, weight, bias


def _aligned(*tensors):
    return all(t is None or (t.data_ptr() % 16 == 0 and (t.dim() == 1 or t.stride(0) * t.element_size() % 16 == 0)) for t in tensors)


def _forward(x, residual, weight, bias, residual_scale, eps, quant, residual_out, out, keep):
    """The launch, after the checks: (residual rows, h, (codes, scales), stats, args, read). ``keep``: stats fp32
    [2, tokens] (mean and rstd) for the backward pass; args: the launch's DgmLayerNormArgs; read: the tensors whose
    memory it names."""
    T, H = x.shape
    read = _readable(x, residual, weight, bias)
    same = residual is None and residual_scale == 1.0 and residual_out is None
    r_out = None if same else residual_out if residual_out is not None else _new_like(x)
    h = out if out is not None else _new_like(x)
    args = _forward_args(*read, residual_scale, eps)
    stats = rows = None
    if keep:
        stats = torch.empty((2, T), dtype=torch.float32, device=x.device)
        at = stats.data_ptr()
        args.mean, args.rstd = at, at + 4 * T
    if r_out is not None:
        args.residual_out, args.residual_out_stride = r_out.data_ptr(), r_out.stride(0)
    args.h, args.h_stride = h.data_ptr(), h.stride(0)
    fused = quant and H % 8 == 0 and _aligned(*read, r_out, h)
    if fused:
        rows = _new_mxfp4(T, H, x.device)
        args.codes, args.scales = rows[0].data_ptr(), rows[1].data_ptr()
    if T > 0:
        if residual_out is not None or out is not None:
            _check_outputs([t for t in (residual_out, out) if t is not None], [t for t in read if t is not None])
        _lib.check(_lib.load().dgm_layer_norm_residual(ctypes.byref(args), _lib.stream()))
        if residual_out is not None or out is not None:
            _lib.written(*(t for t in (residual_out, out) if t is not None))
    if quant and not fused:
        rows = _quantize(h, 1e-30, True, False)[0]
    return x if same else r_out, h, rows, stats, args, read


@functools.lru_cache(maxsize=1024)
def _groups(T, H):
    return _lib.load().dgm_layer_norm_residual_groups(T, H)


def _backward(d_r, d_h, x, residual, weight, bias, forward, needs):
    """The launches of the backward pass, after the checks; forward: DgmLayerNormArgs over the forward call's inputs and
    its mean and rstd."""
    T, H = x.shape
    args = _lib.LayerNormGradArgs(forward)
    if d_r is not None:
        d_r = _rows(d_r)
        args.d_residual_out, args.d_residual_out_stride = d_r.data_ptr(), d_r.stride(0)
    if d_h is not None:
        d_h = _rows(d_h)
        args.d_h, args.d_h_stride = d_h.data_ptr(), d_h.stride(0)
    d_x = d_residual = d_weight = d_bias = None
    if needs[0]:
        d_x = _new_like(x)
        args.d_x, args.d_x_stride = d_x.data_ptr(), H
    if needs[1] and residual is not None:
        d_residual = _new_like(x)
        args.d_residual, args.d_residual_stride = d_residual.data_ptr(), H
    if needs[2] and weight is not None:
        d_weight = _new_like(weight)
        args.d_weight = d_weight.data_ptr()
    if needs[3] and bias is not None:
        d_bias = _new_like(bias)
        args.d_bias = d_bias.data_ptr()
    if d_weight is not None or d_bias is not None:
        ws = torch.empty(2 * _groups(T, H) * H, dtype=torch.float32, device=x.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.nbytes
    _lib.check(_lib.load().dgm_layer_norm_residual_backward(ctypes.byref(args), _lib.stream()))
    return d_x, d_residual, d_weight, d_bias


def _check_backward(d_r, d_h, x, residual, weight, bias, mean, rstd):
    _check(x, residual, weight, bias)
    for d in (d_r, d_h):
        if d is not None and (d.dtype != x.dtype or d.shape != x.shape):
            raise TypeError(f"gradient rows of {x.dtype} {tuple(x.shape)} expected, got {d.dtype} {tuple(d.shape)}")
    for t in (mean, rstd):
        if t is None or t.dtype != torch.float32 or tuple(t.shape) != (x.size(0),) or not t.is_contiguous():
            raise ValueError("mean and rstd of layer_norm_residual_forward (fp32 [tokens]) expected")
    _lib.require_one_device(x, d_r, d_h, residual, weight, bias, mean, rstd)


class _LayerNormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, residual_scale, eps):
        r, h, _, stats, args, read = _forward(x, residual, weight, bias, residual_scale, eps, None, None, None, True)
        saved = x, residual, weight, bias, stats
        ctx.save_for_backward(*saved)
        ctx.options = residual_scale, eps
        # (the launch's arguments, those copies that the kernels read for inputs, and where the saved tensors were)
        ctx.args, ctx.copies, ctx.places = args, [None if u is t else u for t, u in zip(saved, read)], _places(saved)
        ctx.set_materialize_grads(False)
        # (r may be x: autograd hands out an alias of it, whose gradient comes to this backward pass with h's)
        return r, h

    @staticmethod
    def backward(ctx, d_r, d_h):
        _lib.no_second_derivative()
        saved = ctx.saved_tensors
        _lib.no_tangents(d_r, d_h, *saved)
        args = ctx.args
        if _places(saved) != ctx.places:
            # Other memory since the forward pass: storage replaced, or tensors that saved-tensor hooks brought back.
            # What a hook returns is checked as an argument is: the kernels read it by address.
            stats = saved[4].contiguous()
            if stats.dim() != 2 or stats.size(0) != 2:
                raise ValueError(f"saved mean and rstd came back as {tuple(stats.shape)}")
            _check_backward(d_r, d_h, *saved[:4], stats[0], stats[1])
            read = _readable(*saved[:4])
            args = _forward_args(*read, *ctx.options)
            at = stats.data_ptr()
            args.mean, args.rstd = at, at + 4 * stats.size(1)
        return (*_backward(d_r, d_h, *saved[:4], args, ctx.needs_input_grad), None, None)


def layer_norm_residual(x, residual=None, weight=None, bias=None, residual_scale=1.0, eps=1e-5, quant=None,
                        residual_out=None, out=None):
    """The scaled residual add and the layer norm behind it, in one pass over the rows:

        r = residual + residual_scale * x           (r = residual_scale * x without residual)
        h = (r - mean(r)) / sqrt(mean((r - mean(r))^2) + eps) * weight + bias

    x, residual: bf16, fp16 or fp32 [tokens < 2^22, hidden <= 16384], any row stride; weight and bias [hidden] of that
    type or fp32 (both of one). Every part but x may be absent. Arithmetic in fp32 (a row's sum and the squares of its
    differences from the mean have to stay below 3.4e38); r enters the norm unrounded. Returns ``(r, h)``, r x itself
    where nothing changes it (an alias of it under autograd); with ``quant="mxfp4"`` (bf16) ``(r, h, (codes, scales))``:
    the MXFP4 rows of the rounded h (bit for bit ``mxfp4_quantize(h)``), as ``mxfp4_gemm_nt`` takes them.
    ``residual_out`` / ``out``: where r and h go; either may be x's or residual's own rows.

    Differentiable in x, residual, weight and bias (not with quant, residual_out or out; under graph capture use
    ``layer_norm_residual_forward`` and ``layer_norm_residual_backward``). Work runs on the current stream of the
    tensors' device, which has to be the current one."""
    _check(x, residual, weight, bias, quant, residual_out, out)
    _lib.no_tangents(x, residual, weight, bias, residual_out, out)
    _lib.require_one_device(x, residual, weight, bias, residual_out, out)
    residual_scale, eps = float(residual_scale), float(eps)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)
                                    or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)
                                    or (residual_out is not None and residual_out.requires_grad)
                                    or (out is not None and out.requires_grad)):
        _lib.no_graph_under_capture()
        if quant or residual_out is not None or out is not None:
            raise ValueError("quant, residual_out and out have no gradient: call under torch.no_grad()")
        return _LayerNormResidual.apply(x, residual, weight, bias, residual_scale, eps)
    r, h, rows, *_ = _forward(x, residual, weight, bias, residual_scale, eps, quant, residual_out, out, False)
    return (r, h, rows) if quant else (r, h)


def layer_norm_residual_forward(x, residual=None, weight=None, bias=None, residual_scale=1.0, eps=1e-5):
    """``layer_norm_residual`` with what its explicit backward call needs: ``(r, h, mean, rstd)`` (fp32 [tokens] each).
    Records no autograd graph."""
    _check(x, residual, weight, bias)
    _lib.no_tangents(x, residual, weight, bias)
    _lib.require_one_device(x, residual, weight, bias)
    with torch.no_grad():
        r, h, _, stats, _, _ = _forward(x, residual, weight, bias, float(residual_scale), float(eps), None, None, None, True)
    return r, h, stats[0], stats[1]


def layer_norm_residual_backward(d_r, d_h, x, residual, mean, rstd, weight=None, bias=None, residual_scale=1.0, eps=1e-5,
                                 needs=(True,) * 4):
    """Gradients of ``layer_norm_residual``: ``(d_x, d_residual, d_weight, d_bias)`` from d_r = dL/dr and d_h = dL/dh
    (either may be None: zero), the forward call's inputs and the mean and rstd of ``layer_norm_residual_forward``; None
    for an absent input or one that ``needs`` leaves out. r is recomputed in fp32 from x and residual. Sums over tokens
    (weight and bias) are taken in fp32 in a fixed order."""
    _check_backward(d_r, d_h, x, residual, weight, bias, mean, rstd)
    _lib.no_tangents(d_r, d_h, x, residual, weight, bias)
    read = _readable(x, residual, weight, bias)
    forward = _forward_args(*read, float(residual_scale), float(eps))
    forward.mean, forward.rstd = mean.data_ptr(), rstd.data_ptr()
    return _backward(d_r, d_h, x, residual, weight, bias, forward, needs)


__all__ = ["layer_norm_residual", "layer_norm_residual_forward", "layer_norm_residual_backward"]
