"""A decoder block's feed-forward half around the MoE layer, on the GPU (no counterpart in the reference,
whose calls start at the router and end at the combine)."""
import torch

from . import _lib
from .int8_gemm import MAX_K, _operand, int8_gemm_nt
from .mega import mxfp4_mega_moe_from_bf16
from .norm import _check as _check_norm, _forward as _norm
from .quantization_qoq_fused import per_token_cast_to_int8


def mega_moe_block(x, norm_weight, router_weight, l1, l2, sym_buffer, residual=None, shared_expert=None, post_weight=None,
                   gate=None, gate_sigmoid=False, residual_scale=1.0, next_weight=None, eps=1e-6,
                   cumulative_local_expert_recv_stats=None, activation_clamp=10.0, force_balanced=None, token_offset=0,
                   phase_stamps=None, one_launch=None, fast_math=True):
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
    ``sym_buffer`` holds every expert: on an expert-parallel share y is this rank's part of a sum, so such a
    buffer is refused (the parts called one by one, with the sum behind the layer, serve it).
    Returns ``(r, h)``: the new residual stream and, with ``next_weight``, the next norm's output (else
    None). Inference only: under autograd it raises."""
    weights = () if shared_expert is None else tuple(t for pair in shared_expert for t in pair)
    leaves = (x, residual, norm_weight, router_weight, post_weight, gate, next_weight) + weights
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
    residual_scale = float(residual_scale)
    if norm_weight is None:
        raise TypeError("norm_weight: [hidden] expected, got None")
    _check_norm(x, residual, None, norm_weight, None)
    _check_norm(x, None, post_weight, next_weight, gate)
    if weights:
        gate_up, down = _operand("gate and up", shared_expert[0])[0], _operand("down", shared_expert[1])[0]
        inner = down.size(1)
        if tuple(gate_up.shape) != (2 * inner, x.size(1)) or down.size(0) != x.size(1) or inner % 128 or not 0 < inner <= MAX_K:
            raise ValueError(f"shared_expert: gate and up rows [2 I, {x.size(1)}] for down [{x.size(1)}, I], I a multiple of 128 "
                             f"up to {MAX_K}; got {tuple(gate_up.shape)} and {tuple(down.shape)}")
        if activation_clamp is not None and not activation_clamp >= 0:
            raise ValueError(f"activation_clamp {activation_clamp}: at least 0, or None")
    _lib.require_one_device(*leaves)
    with torch.no_grad():
        s, h, q, sf, *_ = _norm(x, residual, None, norm_weight, None, False, 1.0, eps, "int8" if weights else None, None, None,
                                False)
        y = torch.empty_like(h)
        mxfp4_mega_moe_from_bf16(y, h, router_weight, l1, l2, sym_buffer, cumulative_local_expert_recv_stats,
                                 activation_clamp, force_balanced, token_offset, phase_stamps, one_launch)
        if weights and x.size(0):
            act = torch.empty((x.size(0), inner), dtype=torch.bfloat16, device=x.device)
            int8_gemm_nt((q, sf), shared_expert[0], act, activation="swiglu", activation_clamp=activation_clamp)
            int8_gemm_nt(per_token_cast_to_int8(act), shared_expert[1], y, c=y)
        return _norm(y, s, post_weight, next_weight, gate, gate_sigmoid, residual_scale, eps, None, None, None, False)[:2]


__all__ = ["mega_moe_block"]
