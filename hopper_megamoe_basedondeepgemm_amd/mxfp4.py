"""MXFP4 (E2M1 codes with an E8M0 scale for each 32) outside the routed experts, on the GPU: rows and columns of any
matrix quantised, products of such rows, and a linear layer trained on them.

No counterpart in the reference, whose MXFP4 lives in the experts' weights and the activations between them
(deep_gemm/utils/math.py:85 ``per_token_cast_to_fp4`` is the rule of the codes and scales here too)."""
import ctypes
import functools
import math

import torch

from . import _lib

MAX_DIM = 1 << 24


def _rows(t):
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def _fits(m, n):
    return ((m + 63) // 64) * ((n + 63) // 64) < 1 << 23


def _check_quantize(x, amax_floor):
    shape = x.shape
    if x.dtype not in _lib.SRC_DTYPES or len(shape) != 2:
        raise TypeError(f"x must be bf16, fp16 or fp32 [rows, cols], got {x.dtype} {tuple(shape)}")
    if shape[0] >= MAX_DIM or shape[1] >= MAX_DIM:
        raise ValueError(f"x {tuple(shape)}: below 2^24 each way")
    if not 0 <= amax_floor < math.inf:
        raise ValueError(f"amax_floor {amax_floor}: a number, at least 0")


def _new(rows, cols, device):
    """Uninitialised (codes, scales) of rows of cols elements."""
    blocks = (cols + 31) // 32
    return (torch.empty((rows, 16 * blocks), dtype=torch.uint8, device=device),
            torch.empty((rows, blocks), dtype=torch.uint8, device=device))


def _quantize(x, amax_floor, rows, columns):
    """((codes, scales) of x's rows, the same of its columns), each if wanted, after the checks."""
    stride, one = x.stride()
    if one != 1:
        if stride == 1:                                   # (a transposed view: its rows are the memory's columns)
            by_column, by_row = _quantize(x.t(), amax_floor, columns, rows)
            return by_row, by_column
        if x.size(1) != 1:
            x = x.contiguous()
            stride = x.stride(0)
    m, n = x.shape
    by_row = by_column = None
    r = r_sf = c = c_sf = 0
    if rows:
        by_row = _new(m, n, x.device)
        r, r_sf = by_row[0].data_ptr(), by_row[1].data_ptr()
    if columns:
        by_column = _new(n, m, x.device)
        c, c_sf = by_column[0].data_ptr(), by_column[1].data_ptr()
    if m and n:
        args = _lib.Mxfp4QuantArgs(x.data_ptr(), r, r_sf, c, c_sf, m, n, stride, _lib.SRC_DTYPES[x.dtype], amax_floor)
        _lib.check(_lib.load().dgm_mxfp4_quantize(ctypes.byref(args), _lib.stream()))
    return by_row, by_column


def _refuse_gradient(*tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("codes and scales have no gradient: call under torch.no_grad(), or mxfp4_linear")
    _lib.no_tangents(*tensors)


def mxfp4_quantize(x, transpose=False, amax_floor=1e-30):
    """``(codes, scales)`` of x's rows, or with ``transpose`` of its columns, as ``mxfp4_gemm_nt`` takes them:

        block of 32 along a row: e = least integer with max(|block|, amax_floor) <= 6 2^e (at least -126),
        codes = nearest E2M1 of block / 2^e (midpoints to the smaller magnitude), scale byte e + 127

    x: bf16, fp16 or fp32 [rows, cols], any strides, each size below 2^24. codes uint8 [rows, 16 ceil(cols / 32)], two a
    byte, the first in the low half; scales uint8 [rows, ceil(cols / 32)]; behind the last column a block holds zeros.
    (The codes and scale bytes of ``per_token_cast_to_fp4(x, amax_floor=...)``, which takes bf16 rows of whole blocks.)
    A block with an infinity or NaN has scale 255 (NaN) and zeros, so that a product with it is NaN.
    No gradient. Work runs on the current stream of x's device, which has to be the current one."""
    _check_quantize(x, amax_floor)
    _refuse_gradient(x)
    _lib.require_one_device(x)
    return _quantize(x, amax_floor, not transpose, transpose)[1 if transpose else 0]


def mxfp4_quantize_both(x, amax_floor=1e-30):
    """``(mxfp4_quantize(x), mxfp4_quantize(x, transpose=True))`` from one pass over x: what a product along x's columns
    and one along its rows take (a weight in the forward pass and for its input's gradient)."""
    _check_quantize(x, amax_floor)
    _refuse_gradient(x)
    _lib.require_one_device(x)
    return _quantize(x, amax_floor, True, True)


def _operand(name, pair):
    """(codes, scale bytes, rows, bytes of a code row) of a product's operand."""
    q, sf = pair
    shape, sf_shape = q.shape, sf.shape
    if q.dtype != torch.uint8 or len(shape) != 2:
        raise TypeError(f"{name}: uint8 codes [rows, k / 2] expected, got {q.dtype} {tuple(shape)}")
    if sf.dtype == torch.int32 and len(sf_shape) == 2:         # (per_token_cast_to_fp4(use_packed_ue8m0=True))
        sf = sf.contiguous().view(torch.uint8)
        sf_shape = sf.shape
    rows, size = shape
    if sf.dtype != torch.uint8 or len(sf_shape) != 2 or sf_shape[0] != rows or size != 16 * sf_shape[1]:
        raise TypeError(f"{name}: uint8 scales [{rows}, {size / 16:g}] (a byte for 16 bytes of codes) expected, got "
                        f"{sf.dtype} {tuple(sf_shape)}")
    return q, sf, rows, size


def _readable(q, sf):
    """An operand as the kernels read it, code rows on 16 bytes and less than 2^23 apart, scale rows of contiguous bytes:
    (codes, scales, their addresses, their row strides)."""
    stride, one = q.stride()
    at = q.data_ptr()
    if one != 1 or stride % 16 or stride >= 1 << 23 or at % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        stride, at = q.stride(0), q.data_ptr()
    sf_stride, one = sf.stride()
    if one != 1 and sf.size(1) != 1:
        sf = sf.contiguous()
        sf_stride = sf.stride(0)
    return q, sf, at, sf.data_ptr(), stride, sf_stride


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(m, n, k, swiglu):
    return _lib.load().dgm_mxfp4_gemm_workspace_bytes(m, n, k, int(swiglu))


def mxfp4_gemm_nt(a, b, d, c=None, activation=None, activation_clamp=10.0, fast_math=True):
    """d = a @ b.T over MXFP4 rows, into d (bf16, fp16 or fp32 [m, n], any row stride):

        d[m, n] = sum over blocks 2^(sa + sb - 254) sum of code products (+ c[m, n], or c[n] for a 1-D c)

    a = (codes [m, k / 2], scales [m, k / 32]) and b of n rows, as ``mxfp4_quantize`` returns them for tokens and
    weights (or ``per_token_cast_to_fp4`` with ``use_packed_ue8m0``; the two halves of a byte have to be in one order in
    both). c has d's type and may be d itself. ``activation="swiglu"``: b holds gate rows, then up rows, and
    d [m, n / 2] = silu(min(gate, clamp)) * clamp(up, -clamp, clamp), the layer's SwiGLU (``activation_clamp`` None: no
    clamp; ``fast_math`` as in ``int8_gemm_nt``). Sums in fp32, one rounding; a scale of 255 makes its row NaN. k a
    multiple of 32. m, n and k below 2^24, ceil(m / 64) ceil(n / 64) below 2^23. No gradient (``mxfp4_linear`` has
    one). Work runs on the current stream of the tensors' device, which has to be the current one. Returns d."""
    aq, asf, m, size_a = _operand("a", a)
    bq, bsf, n, size_b = _operand("b", b)
    k = 2 * size_a
    if size_a != size_b or not 32 <= k < MAX_DIM:
        raise ValueError(f"k of a {k} and of b {2 * size_b}: equal, 32 to 2^24")
    if activation not in (None, "swiglu"):
        raise ValueError(f"activation {activation!r}: None or 'swiglu'")
    swiglu = activation is not None
    if swiglu and (n % 2 or c is not None):
        raise ValueError("swiglu takes a gate and an up half of b's rows, and no c")
    if activation_clamp is not None and not activation_clamp >= 0:
        raise ValueError(f"activation_clamp {activation_clamp}: at least 0, or None")
    if m >= MAX_DIM or n >= MAX_DIM or not _fits(m, n):
        raise ValueError(f"m {m} and n {n}: below 2^24, and ceil(m / 64) ceil(n / 64) below 2^23")
    n_out = n // 2 if swiglu else n
    dtype = _lib.SRC_DTYPES.get(d.dtype)
    if dtype is None or d.shape != (m, n_out):
        raise TypeError(f"d: bf16, fp16 or fp32 [{m}, {n_out}] expected, got {d.dtype} {tuple(d.shape)}")
    d_stride, one = d.stride()
    if m and n_out and ((n_out > 1 and one != 1) or (m > 1 and d_stride < n_out)):
        raise ValueError("d: rows must be contiguous and must not overlap")
    if c is not None and (c.dtype != d.dtype or tuple(c.shape) not in ((m, n_out), (n_out,))):
        raise TypeError(f"c: {d.dtype} [{m}, {n_out}] or [{n_out}] expected, got {c.dtype} {tuple(c.shape)}")
    if (d.requires_grad or (c is not None and c.requires_grad)) and torch.is_grad_enabled():
        raise RuntimeError("mxfp4_gemm_nt has no gradient: call it under torch.no_grad(), or mxfp4_linear")
    _lib.no_tangents(d, c)
    _lib.require_one_device(d, aq, asf, bq, bsf, c)
    if m == 0 or n_out == 0:
        return d
    aq, asf, pa, psa, a_stride, sa_stride = _readable(aq, asf)
    bq, bsf, pb, psb, b_stride, sb_stride = _readable(bq, bsf)
    size, lo, last = 2 if dtype < 2 else 4, d.data_ptr(), m - 1
    hi = lo + (last * d_stride + n_out) * size
    if ((pa < hi and lo < pa + last * a_stride + size_a) or (pb < hi and lo < pb + (n - 1) * b_stride + size_b)
            or (psa < hi and lo < psa + last * sa_stride + size_a // 16) or (psb < hi and lo < psb + (n - 1) * sb_stride + size_b // 16)):
        raise ValueError("d overlaps an operand")
    args = _lib.Mxfp4GemmArgs(pa, psa, pb, psb, 0, lo, m, n, k, a_stride, sa_stride, b_stride, sb_stride, 0, d_stride,
                              dtype, swiglu, math.inf if activation_clamp is None else float(activation_clamp),
                              1 if fast_math else 0)
    if c is not None:
        if c.dim() == 1:
            c, c_stride, end = c.contiguous(), 0, n_out
        else:
            c = _rows(c)
            c_stride = c.stride(0)
            end = last * c_stride + n_out
        pc = c.data_ptr()
        if pc < hi and lo < pc + end * size and not (pc == lo and c.dim() == 2 and (m == 1 or c_stride == d_stride)):
            raise ValueError("c overlaps d other than as the same rows")
        args.c, args.c_stride = pc, c_stride
    need = _workspace_bytes(m, n, k, swiglu)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=d.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _lib.check(_lib.load().dgm_mxfp4_gemm_nt(ctypes.byref(args), _lib.stream()))
    _lib.written(d)
    return d


def _check_linear(x, weight):
    _check_quantize(x, 0.0)
    if weight.dtype not in _lib.SRC_DTYPES or weight.dim() != 2 or weight.size(1) != x.size(1):
        raise TypeError(f"weight must be bf16, fp16 or fp32 [out, {x.size(1)}], got {weight.dtype} {tuple(weight.shape)}")
    (m, k), n = x.shape, weight.size(0)
    if k == 0 or n == 0:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)}: no feature")
    if n >= MAX_DIM or not (_fits(m, n) and _fits(m, k) and _fits(n, k)):
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)}: sizes below 2^24, and ceil(a / 64) ceil(b / 64) below "
                         "2^23 for each two of tokens, in and out")


@functools.lru_cache(maxsize=1024)
def _linear_workspace_bytes(m, n, k, backward):
    return _lib.load().dgm_mxfp4_linear_workspace_bytes(m, n, k, backward)


def _code_bytes(rows, cols):
    return rows * 16 * ((cols + 31) // 32)


def _columns_memory(rows, cols, like):
    """One piece of memory for the codes and scales of rows of cols elements."""
    return torch.empty(_code_bytes(rows, cols) // 16 * 17, dtype=torch.uint8, device=like.device)


def _as_pair(memory, rows, cols):
    codes, blocks = _code_bytes(rows, cols), (cols + 31) // 32
    return memory[:codes].view(rows, 16 * blocks), memory[codes:].view(rows, blocks)


def _linear_forward(x, weight, keep_x, keep_weight):
    """y, what the weight's gradient needs (x's columns) and what x's needs (the weight's columns), if wanted."""
    x, weight = _rows(x), _rows(weight)
    (m, k), n = x.shape, weight.size(0)
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    args = _lib.Mxfp4LinearArgs(x=x.data_ptr(), w=weight.data_ptr(), y=y.data_ptr(), m=m, n=n, k=k, x_stride=x.stride(0),
                                w_stride=weight.stride(0), x_dtype=_lib.SRC_DTYPES[x.dtype], w_dtype=_lib.SRC_DTYPES[weight.dtype])
    xt = wt = None
    if keep_x:
        xt = _columns_memory(k, m, x)
        if m:
            at = xt.data_ptr()
            args.x_columns, args.x_column_scales = at, at + _code_bytes(k, m)
    if keep_weight:
        wt = _columns_memory(k, n, x)
        at = wt.data_ptr()
        args.w_columns, args.w_column_scales = at, at + _code_bytes(k, n)
    if m:
        need = _linear_workspace_bytes(m, n, k, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _lib.check(_lib.load().dgm_mxfp4_linear(ctypes.byref(args), _lib.stream()))
    return y, xt, wt


def _linear_backward(d_y, xt, wt, k, x_dtype, w_dtype):
    """(d_x, d_weight), each where its operand (addresses of codes and scales) is given."""
    d_y = _rows(d_y)
    m, n = d_y.shape
    args = _lib.Mxfp4LinearArgs(d_y=d_y.data_ptr(), m=m, n=n, k=k, d_y_stride=d_y.stride(0), x_dtype=_lib.SRC_DTYPES[x_dtype],
                                w_dtype=_lib.SRC_DTYPES[w_dtype])
    d_x = d_w = None
    if wt is not None:
        d_x = torch.empty((m, k), dtype=x_dtype, device=d_y.device)
        args.d_x = d_x.data_ptr()
        args.w_columns, args.w_column_scales = wt
    if xt is not None:
        d_w = torch.empty((n, k), dtype=w_dtype, device=d_y.device)
        if m == 0:
            d_w.zero_()                    # (a sum over no tokens)
        else:
            args.d_w = d_w.data_ptr()
            args.x_columns, args.x_column_scales = xt
    if m:
        need = _linear_workspace_bytes(m, n, k, 1)
        ws = torch.empty(need, dtype=torch.uint8, device=d_y.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
        _lib.check(_lib.load().dgm_mxfp4_linear_backward(ctypes.byref(args), _lib.stream()))
    return d_x, d_w


class _Mxfp4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        y, xt, wt = _linear_forward(x, weight, ctx.needs_input_grad[1], ctx.needs_input_grad[0])
        ctx.save_for_backward(xt, wt)
        ctx.shape = x.size(0), weight.size(0), x.size(1), x.dtype, weight.dtype
        return y

    @staticmethod
    def backward(ctx, d_y):
        _lib.no_second_derivative()
        saved = ctx.saved_tensors
        _lib.no_tangents(d_y, *saved)
        m, n, k, x_dtype, w_dtype = ctx.shape
        kept = []
        for memory, wanted, inner in ((saved[0], ctx.needs_input_grad[1], m), (saved[1], ctx.needs_input_grad[0], n)):
            if not wanted:
                kept.append(None)
                continue
            # (what saved-tensor hooks bring back is checked as an argument is: the kernels read it by address)
            size = _code_bytes(k, inner)
            if memory.dtype != torch.uint8 or tuple(memory.shape) != (size // 16 * 17,):
                raise ValueError(f"saved columns came back as {memory.dtype} {tuple(memory.shape)}")
            kept.append((_contiguous16(memory), size))
        _lib.require_one_device(d_y, *(p[0] for p in kept if p is not None))
        at = [None if p is None else (p[0].data_ptr(), p[0].data_ptr() + p[1]) for p in kept]
        return _linear_backward(d_y, *at, k, x_dtype, w_dtype)


def mxfp4_linear(x, weight):
    """y = x @ weight.T with all three products of a training step in MXFP4:

        y = q(x) q(weight)^T,  d_x = q(d_y) q(weight^T)^T,  d_weight = q(d_y^T) q(x^T)^T

    q as ``mxfp4_quantize`` along the dimension that its product sums over; the gradients pass straight through the
    roundings. x: bf16, fp16 or fp32 [tokens, in], weight: any of them [out, in] (fp32 master weights); y and d_x have
    x's type, d_weight the weight's; any strides, each size below 2^24, products within ``mxfp4_gemm_nt``'s limits.
    The backward pass keeps the codes of x's and the weight's columns (17 / 32 byte a value), not the inputs. Under graph
    capture use ``mxfp4_linear_forward`` and ``mxfp4_linear_backward``. Work runs on the current stream of the tensors'
    device, which has to be the current one."""
    _check_linear(x, weight)
    _lib.no_tangents(x, weight)
    _lib.require_one_device(x, weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        _lib.no_graph_under_capture()
        return _Mxfp4Linear.apply(x, weight)
    return _linear_forward(x, weight, False, False)[0]


def mxfp4_linear_forward(x, weight, needs=(True, True)):
    """``mxfp4_linear`` with what its explicit backward call needs: ``(y, x_columns, weight_columns)`` (each
    ``mxfp4_quantize(..., transpose=True)`` of its input; None where ``needs`` of (d_x, d_weight) does not want it).
    Records no autograd graph."""
    _check_linear(x, weight)
    _lib.no_tangents(x, weight)
    _lib.require_one_device(x, weight)
    with torch.no_grad():
        y, xt, wt = _linear_forward(x, weight, bool(needs[1]), bool(needs[0]))
    k = x.size(1)
    return y, None if xt is None else _as_pair(xt, k, x.size(0)), None if wt is None else _as_pair(wt, k, weight.size(0))


def mxfp4_linear_backward(d_y, x_columns, weight_columns, x_shape, weight_shape, weight_dtype=None, needs=(True, True)):
    """Gradients of ``mxfp4_linear``: ``(d_x, d_weight)`` from d_y = dL/dy and what ``mxfp4_linear_forward`` returned for
    x of x_shape and the weight of weight_shape; d_x has d_y's type, d_weight ``weight_dtype`` (None: d_y's). None for
    what ``needs`` leaves out."""
    weight_dtype = weight_dtype or d_y.dtype
    if d_y.dtype not in _lib.SRC_DTYPES or weight_dtype not in _lib.SRC_DTYPES:
        raise TypeError(f"d_y and the weight are bf16, fp16 or fp32, got {d_y.dtype} and {weight_dtype}")
    if len(x_shape) != 2 or len(weight_shape) != 2 or x_shape[1] != weight_shape[1] or x_shape[1] < 1 or weight_shape[0] < 1:
        raise ValueError(f"x {tuple(x_shape)} and weight {tuple(weight_shape)}: [tokens, in] and [out, in]")
    (m, k), n = x_shape, weight_shape[0]
    if max(m, n, k) >= MAX_DIM or not (_fits(m, k) and _fits(n, k)):
        raise ValueError(f"x {tuple(x_shape)} and weight {tuple(weight_shape)}: sizes below 2^24, and ceil(a / 64) ceil(b / 64) below 2^23")
    if tuple(d_y.shape) != (m, n):
        raise TypeError(f"d_y [{m}, {n}] expected, got {tuple(d_y.shape)}")
    kept = []
    for name, pair, wanted, inner in (("x_columns", x_columns, needs[1], m), ("weight_columns", weight_columns, needs[0], n)):
        if not wanted:
            kept.append(None)
            continue
        blocks = (inner + 31) // 32
        if pair is None or any(t.dtype != torch.uint8 for t in pair) or tuple(pair[0].shape) != (k, 16 * blocks) \
                or tuple(pair[1].shape) != (k, blocks):
            raise ValueError(f"{name}: uint8 codes [{k}, {16 * blocks}] and scales [{k}, {blocks}] expected, as mxfp4_linear_forward "
                             "returns them")
        kept.append(pair)
    _lib.no_tangents(d_y)
    _lib.require_one_device(d_y, *(t for pair in kept if pair is not None for t in pair))
    # (the tensors are held until the launches are enqueued)
    kept = [None if p is None else (_contiguous16(p[0]), p[1].contiguous()) for p in kept]
    at = [None if p is None else (p[0].data_ptr(), p[1].data_ptr()) for p in kept]
    with torch.no_grad():
        return _linear_backward(d_y, *at, k, d_y.dtype, weight_dtype)


def _contiguous16(t):
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


__all__ = ["mxfp4_quantize", "mxfp4_quantize_both", "mxfp4_gemm_nt", "mxfp4_linear", "mxfp4_linear_forward",
           "mxfp4_linear_backward"]
