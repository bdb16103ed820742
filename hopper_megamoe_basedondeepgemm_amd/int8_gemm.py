"""int8 products with a scale for each token and channel, on the GPU: the dense (shared) expert beside
the routed ones, on the int8 rows that ``per_token_cast_to_int8`` and ``rms_norm_residual`` write."""
import ctypes
import functools
import math

import torch

from . import _lib

MAX_K = 131071          # sums of K products of up to 128 * 128 stay below 2^31


def _operand(name, pair):
    """(int8 rows, fp32 scales): scales [rows], or one scale per row repeated [rows, groups] as
    ``per_token_cast_to_int8`` returns them (the first column is read; comparing it with the last one in the kernel
    took 4 to 6 % of a decode call, those with one scale a row too)."""
    q, sf = pair
    if q.dtype != torch.int8 or q.dim() != 2:
        raise TypeError(f"{name}: int8 [rows, k] expected, got {q.dtype} {tuple(q.shape)}")
    if sf.dtype != torch.float32 or sf.dim() not in (1, 2) or sf.size(0) != q.size(0) or (sf.dim() == 2 and sf.size(1) < 1):
        raise TypeError(f"{name}: fp32 scales [{q.size(0)}] (or repeated [{q.size(0)}, groups]) expected, got {sf.dtype} "
                        f"{tuple(sf.shape)}")
    return q, sf


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(m, n, k, swiglu):
    return _lib.load().dgm_int8_gemm_workspace_bytes(m, n, k, int(swiglu))


def _rows(t):
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def int8_gemm_nt(a, b, d, c=None, activation=None, activation_clamp=10.0, fast_math=True):
    """d = (a @ b.T) with a scale for each row of both, into d (bf16, fp16 or fp32 [m, n], any row stride):

        d[m, n] = sfa[m] * sfb[n] * sum_k a[m, k] * b[n, k] (+ c[m, n], or c[n] for a 1-D c)

    a = (int8 [m, k], fp32 scales), b = (int8 [n, k], fp32 scales); scales [rows], or repeated per row as
    ``per_token_cast_to_int8`` returns them (it also packs the weights: one scale per channel). Of repeated scales
    the first column is read, without a look at the others: scales that differ over groups of k are another product,
    which this is not. sfa[m] * sfb[n] is taken first and has to be zero or a normal fp32 number. c has d's type and
    may be d itself. ``activation="swiglu"``: b holds gate rows, then up rows, and d [m, n / 2] = silu(min(gate,
    clamp)) * clamp(up, -clamp, clamp), the layer's SwiGLU (``activation_clamp`` None: no clamp; ``fast_math`` as in
    ``mxfp4_mega_moe_fused``; unlike the layer's it keeps NaN, of scales that are infinite or NaN). Sums are exact
    in int32 (k <= 131071), the rest is fp32, rounded once. 16-byte aligned rows (k a multiple of 16) take the fast kernels. No gradient. Work
    runs on the current stream of the tensors' device, which has to be the current one. Returns d."""
    aq, asf = _operand("a", a)
    bq, bsf = _operand("b", b)
    m, k = aq.shape
    n = bq.size(0)
    if bq.size(1) != k or not 1 <= k <= MAX_K:
        raise ValueError(f"k of a {k} and of b {bq.size(1)}: equal, 1 to {MAX_K}")
    if activation not in (None, "swiglu"):
        raise ValueError(f"activation {activation!r}: None or 'swiglu'")
    swiglu = activation is not None
    if swiglu and (n % 2 or c is not None):
        raise ValueError("swiglu takes a gate and an up half of b's rows, and no c")
    if activation_clamp is not None and not activation_clamp >= 0:
        raise ValueError(f"activation_clamp {activation_clamp}: at least 0, or None")
    if m >= 1 << 20 or n >= 1 << 24:
        raise ValueError(f"m {m} and n {n}: below 2^20 and 2^24")
    n_out = n // 2 if swiglu else n
    if d.dtype not in _lib.SRC_DTYPES or d.dim() != 2 or d.size(0) != m or d.size(1) != n_out:
        raise TypeError(f"d: bf16, fp16 or fp32 [{m}, {n_out}] expected, got {d.dtype} {tuple(d.shape)}")
    d_stride = d.stride(0)
    if m and n_out and ((n_out > 1 and d.stride(1) != 1) or (m > 1 and d_stride < n_out)):
        raise ValueError("d: rows must be contiguous and must not overlap")
    if c is not None and (c.dtype != d.dtype or tuple(c.shape) not in ((m, n_out), (n_out,))):
        raise TypeError(f"c: {d.dtype} [{m}, {n_out}] or [{n_out}] expected, got {c.dtype} {tuple(c.shape)}")
    if (d.requires_grad or asf.requires_grad or bsf.requires_grad
            or (c is not None and c.requires_grad)) and torch.is_grad_enabled():
        raise RuntimeError("int8_gemm_nt has no gradient: call it under torch.no_grad()")
    _lib.no_tangents(d, asf, bsf, c)
    _lib.require_one_device(d, aq, asf, bq, bsf, c)
    if m == 0 or n_out == 0:
        return d
    aq, bq = _rows(aq), _rows(bq)
    size = d.element_size()
    pa, pb, lo, a_stride, b_stride = aq.data_ptr(), bq.data_ptr(), d.data_ptr(), aq.stride(0), bq.stride(0)
    psa, psb, sa_stride, sb_stride = asf.data_ptr(), bsf.data_ptr(), asf.stride(0), bsf.stride(0)
    hi = lo + ((m - 1) * d_stride + n_out) * size
    if ((pa < hi and lo < pa + (m - 1) * a_stride + k) or (pb < hi and lo < pb + (n - 1) * b_stride + k)
            or (psa < hi and lo < psa + 4 * (m - 1) * sa_stride + 4) or (psb < hi and lo < psb + 4 * (n - 1) * sb_stride + 4)):
        raise ValueError("d overlaps an operand")
    args = _lib.Int8GemmArgs(pa, psa, pb, psb, 0, lo, m, n, k, a_stride, sa_stride, b_stride, sb_stride, 0, d_stride, _lib.SRC_DTYPES[d.dtype], swiglu,
                             math.inf if activation_clamp is None else float(activation_clamp), 1 if fast_math else 0)
    if c is not None:
        if c.dim() == 1:
            c, c_stride, end = c.contiguous(), 0, n_out
        else:
            c = _rows(c)
            c_stride = c.stride(0)
            end = (m - 1) * c_stride + n_out
        pc = c.data_ptr()
        if pc < hi and lo < pc + end * size and not (pc == lo and c.dim() == 2 and (m == 1 or c_stride == d_stride)):
            raise ValueError("c overlaps d other than as the same rows")
        args.c, args.c_stride = pc, c_stride
    need = _workspace_bytes(m, n, k, swiglu)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=d.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _lib.check(_lib.load().dgm_int8_gemm_nt(ctypes.byref(args), _lib.stream()))
    _lib.written(d)
    return d


__all__ = ["int8_gemm_nt"]
