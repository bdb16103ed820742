"""A decoder block's feed-forward half around the MoE layer, on the GPU (no counterpart in the reference,
whose calls start at the router and end at the combine)."""
import torch

from . import _lib
from .int8_gemm import MAX_K, _operand, int8_gemm_nt
from .layer_norm import _check as _check_layer_norm, _forward as _layer_norm
from .mega import mxfp4_mega_moe_from_bf16
from .mxfp4 import MAX_DIM, _fits, _operand as _mxfp4_operand, _quantize as _mxfp4_rows, mxfp4_gemm_nt
from .norm import _check as _check_norm, _forward as _norm
from .quantization_qoq_fused import per_token_cast_to_int8


def mega_moe_block(x, norm_weight, router_weight, l1, l2, sym_buffer, residual=None, shared_expert=None, post_weight=None,
                   gate=None, gate_sigmoid=False, residual_scale=1.0, next_weight=None, eps=1e-6,
                   cumulative_local_expert_recv_stats=None, activation_clamp=10.0, force_balanced=None, token_offset=0,
                   phase_stamps=None, one_launch=None, fast_math=True, norm="rms", norm_bias=None, next_bias=None):
    """Norm, MoE layer with an optional dense expert beside it, and the way back into the residual stream:

        s, h  = rms_norm_residual(x, residual, pre_weight=norm_weight)       (s = residual + x, or x)
        y     = mxfp4_mega_moe_from_bf16(h, ...) on ``sym_buffer`` (with the options from activation_clamp to
                one_launch; its SwiGLU, like the dense expert's, is the fast_math one, so False is refused)
        y    += down(swiglu(gate_up(h)))                                      (shared_expert)
        return rms_norm_residual(y, s, post_weight, next_weight, gate, gate_sigmoid, residual_scale)

    x, residual: bf16 [tokens, hidden] (the block before's output and the residual stream it is added to).
    ``shared_expert = ((int8 [2 I, hidden], scales), (int8 [hidden, I], scales))``: gate rows then up rows, and
    down, each as ``per_token_cast_to_int8`` packs bf16 weights (one scale per channel, I a multiple of
    128); its products are int8 (``int8_gemm_nt``) on the rows that the first norm writes beside h and on
    the cast of the SwiGLU output, and the down product adds to the experts' output in fp32, rounded once.
    Or in the routed experts' own format, each pair as ``mxfp4_quantize`` packs weights (uint8 codes [2 I, hidden / 2]
    and [hidden, I / 2] with their scales; hidden and I multiples of 32): the products are then ``mxfp4_gemm_nt`` on the
    MXFP4 rows of h and of the SwiGLU output.
    ``norm="layer"``: both norms are ``layer_norm_residual`` with norm_bias and next_bias (either may be absent), the way
    back r = s + residual_scale * y; such blocks have no post norm and no gate.
    ``sym_buffer`` holds every expert: on an expert-parallel share y is this rank's part of a sum, so such a
    buffer is refused (the parts called one by one, with the sum behind the layer, serve it).
    Returns ``(r, h)``: the new residual stream and, with ``next_weight``, the next norm's output (else
    None). Inference only: under autograd it raises."""
    weights = () if shared_expert is None else tuple(t for pair in shared_expert for t in pair)
    leaves = (x, residual, norm_weight, router_weight, post_weight, gate, next_weight, norm_bias, next_bias) + weights
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves):
        raise RuntimeError("mega_moe_block has no gradient: call it under torch.no_grad()")
    _lib.no_tangents(*leaves)
    if x.dim() != 2 or x.dtype != torch.bfloat16 or x.size(1) != sym_buffer.hidden:
        raise TypeError(f"x must be bf16 [tokens, {sym_buffer.hidden}], got {x.dtype} {tuple(x.shape)}")
    if sym_buffer.num_local_experts != sym_buffer.num_experts:
        raise ValueError(f"mega_moe_block needs every expert: this buffer's layer computes {sym_buffer.num_local_experts} of "
                         f"{sym_buffer.num_experts}, and what follows it here belongs behind the sum over ranks")
    if not fast_math:
        raise ValueError("fast_math=False: the layer's call from bf16 rows has no IEEE SwiGLU")
    # (all of the block's own arguments: the layer counts its tokens, so nothing may be refused behind it)
    residual_scale, eps = float(residual_scale), float(eps)
    if norm_weight is None:
        raise TypeError("norm_weight: [hidden] expected, got None")
    if norm not in ("rms", "layer"):
        raise ValueError(f"norm {norm!r}: 'rms' or 'layer'")
    layer = norm == "layer"
    if layer:
        if post_weight is not None or gate is not None:
            raise ValueError("norm='layer' has no post_weight and no gate")
        if next_bias is not None and next_weight is None:
            raise ValueError("next_bias without a next_weight")
        _check_layer_norm(x, residual, norm_weight, norm_bias)
        _check_layer_norm(x, None, next_weight, next_bias)
    else:
        if norm_bias is not None or next_bias is not None:
            raise ValueError("norm_bias and next_bias belong to norm='layer'")
        _check_norm(x, residual, None, norm_weight, None)
        _check_norm(x, None, post_weight, next_weight, gate)
    mxfp4 = bool(weights) and shared_expert[0][0].dtype == shared_expert[1][0].dtype == torch.uint8
    if weights:
        operand, unit, least, most = (_mxfp4_operand, 2, 32, MAX_DIM // 2 - 32) if mxfp4 else (_operand, 1, 128, MAX_K)
        gate_up, down = operand("gate and up", shared_expert[0])[0], operand("down", shared_expert[1])[0]
        inner = unit * down.size(1)
        if tuple(gate_up.shape) != (2 * inner, x.size(1) // unit) or x.size(1) % unit or down.size(0) != x.size(1) or inner % least \
                or not 0 < inner <= most:
            raise ValueError(f"shared_expert: gate and up rows [2 I, {x.size(1)}] for down [{x.size(1)}, I], I a multiple of {least} "
                             f"up to {most}; got {tuple(gate_up.shape)} and {tuple(down.shape)}" + (" (two codes a byte)" if mxfp4 else ""))
        if mxfp4 and not (_fits(x.size(0), 2 * inner) and _fits(x.size(0), x.size(1))):
            raise ValueError(f"shared_expert of {inner} channels for x {tuple(x.shape)}: ceil(tokens / 64) ceil(rows / 64) below 2^23 "
                             "for both weights' rows")
        if activation_clamp is not None and not activation_clamp >= 0:
            raise ValueError(f"activation_clamp {activation_clamp}: at least 0, or None")
    _lib.require_one_device(*leaves)
    with torch.no_grad():
        if layer:
            s, h, rows, *_ = _layer_norm(x, residual, norm_weight, norm_bias, 1.0, eps, "mxfp4" if mxfp4 else None, None, None, False)
            if weights and not mxfp4 and x.size(0):
                rows = per_token_cast_to_int8(h)
        else:
            s, h, q, sf, *_ = _norm(x, residual, None, norm_weight, None, False, 1.0, eps, "int8" if weights and not mxfp4 else None,
                                    None, None, False)
            rows = _mxfp4_rows(h, 1e-30, True, False)[0] if mxfp4 else (q, sf)
        y = torch.empty_like(h)
        mxfp4_mega_moe_from_bf16(y, h, router_weight, l1, l2, sym_buffer, cumulative_local_expert_recv_stats,
                                 activation_clamp, force_balanced, token_offset, phase_stamps, one_launch)
        if weights and x.size(0):
            act = torch.empty((x.size(0), inner), dtype=torch.bfloat16, device=x.device)
            if mxfp4:
                mxfp4_gemm_nt(rows, shared_expert[0], act, activation="swiglu", activation_clamp=activation_clamp)
                mxfp4_gemm_nt(_mxfp4_rows(act, 1e-30, True, False)[0], shared_expert[1], y, c=y)
            else:
                int8_gemm_nt(rows, shared_expert[0], act, activation="swiglu", activation_clamp=activation_clamp)
                int8_gemm_nt(per_token_cast_to_int8(act), shared_expert[1], y, c=y)
        if not layer:
            return _norm(y, s, post_weight, next_weight, gate, gate_sigmoid, residual_scale, eps, None, None, None, False)[:2]
        if next_weight is None:                                # (the residual add alone)
            return _norm(y, s, None, None, None, False, residual_scale, eps, None, None, None, False)[0], None
        return _layer_norm(y, s, next_weight, next_bias, residual_scale, eps, None, None, None, False)[:2]


__all__ = ["mega_moe_block"]
