"""The MXFP4 operators and layer norm around the MoE layer that are timed: one pass of each case through the public
entry points.

  norm        residual add and layer norm (``layer_norm_residual``); with "train" the backward pass too
  norm_gemm   the same with MXFP4 rows for the dense expert, and their product with its weights
  quant_gemm  bf16, fp16 or fp32 rows to MXFP4 (``mxfp4_quantize``) and their product with MXFP4 weights
  gemm        MXFP4 rows times MXFP4 weights (``mxfp4_gemm_nt``): plain, added to C or a bias, or with SwiGLU
  linear      a training step of a linear layer whose three products are MXFP4 (``mxfp4_linear``)

With ``own`` false, ``run`` computes the same in elementary torch operations, in 32 bits (column sums over tokens in
64). ``exact`` restates the operators in 64 bits, the norm's gradients by differentiation.
"""
import math

import torch

own = False
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS, CLAMP, FLOOR = 1e-5, 10.0, 1e-30


def _norm(name, rows, hidden, dtype="bf16", wdtype="bf16", residual=True, bias=True, scale=1.0, train=False):
    return {"name": name, "kind": "norm", "rows": rows, "hidden": hidden, "dtype": dtype, "wdtype": wdtype, "residual": residual,
            "bias": bias, "scale": scale, "train": train}


def _gemm(name, m, n, k, out="bf16", add="none", swiglu=False):
    return {"name": name, "kind": "gemm", "m": m, "n": n, "k": k, "out": out, "add": add, "swiglu": swiglu}


def listed():
    return [
        # one sequence being decoded: residual add and the norm before the layer
        _norm("norm-m1-h4096", 1, 4096),
        # a prefill chunk of the same
        _norm("norm-m8192-h4096", 8192, 4096, scale=0.5),
        # a training step with fp32 norm weights
        _norm("norm-train-m4096-h4096", 4096, 4096, wdtype="fp32", train=True),
        # a ragged training batch in fp32, no residual stream (a norm on queries or embeddings)
        _norm("norm-train-m777-h2880-fp32", 777, 2880, dtype="fp32", wdtype="fp32", residual=False, train=True),
        # a decode batch into the dense expert: norm, MXFP4 rows, product
        {"name": "norm-gemm-m64-h7168-n4096", "kind": "norm_gemm", "rows": 64, "hidden": 7168, "n": 4096},
        # a prefill chunk into a narrow projection: the rows' quantisation is most of it
        {"name": "quant-gemm-m8192-n512-k7168", "kind": "quant_gemm", "m": 8192, "n": 512, "k": 7168, "dtype": "bf16"},
        # single token, down projection of the dense expert added to the experts' output
        _gemm("gemm-m1-n4096-k2048-add", 1, 4096, 2048, add="matrix"),
        # a ragged decode batch, gate and up projection with SwiGLU
        _gemm("gemm-m37-n8192-k4096-swiglu", 37, 8192, 4096, swiglu=True),
        # an odd prefill chunk with a bias, fp16 out, K that ends inside the kernels' steps
        _gemm("gemm-m1000-n5120-k2880-bias-fp16", 1000, 5120, 2880, out="fp16", add="bias"),
        # the largest single product: a prefill of 8192 tokens
        _gemm("gemm-m8192-n8192-k4096", 8192, 8192, 4096),
        # a training step of a linear layer: forward, input's and weight's gradient
        {"name": "linear-train-m8192-n4096-k4096", "kind": "linear", "m": 8192, "n": 4096, "k": 4096, "dtype": "bf16", "wdtype": "bf16"},
        # the same with a ragged batch, an odd width and fp32 master weights
        {"name": "linear-train-m777-n1234-k2880-fp32w", "kind": "linear", "m": 777, "n": 1234, "k": 2880, "dtype": "bf16", "wdtype": "fp32"},
    ]


def draw(rng):
    log_int = lambda lo, hi: min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))
    kind = rng.choice(["norm", "norm", "gemm", "gemm", "quant_gemm", "linear", "norm_gemm"])
    if kind == "norm":
        hidden = log_int(256, 8192)
        hidden = hidden if rng.random() < 0.2 else max(8, hidden // 8 * 8)
        rows = log_int(1, max(1, min(8192, 8192 * 4096 // hidden)))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = _norm("", rows, hidden, dtype, rng.choice([dtype, "fp32"]), rng.random() < 0.7, rng.random() < 0.7, rng.choice([1.0, 0.5, 0.22]),
                  rows <= 4096 and rng.random() < 0.5)
    elif kind == "gemm":
        n, k = log_int(256, 8192) // 2 * 2, log_int(256, 8192) // 32 * 32
        m = log_int(1, max(1, min(8192, 8192 * 8192 * 4096 // (n * k))))
        swiglu = rng.random() < 0.3
        c = _gemm("", m, n, k, rng.choice(["bf16", "bf16", "fp16", "fp32"]), "none" if swiglu else rng.choice(["none", "matrix", "bias"]), swiglu)
    elif kind == "quant_gemm":
        c = {"kind": kind, "m": log_int(1, 8192), "n": log_int(64, 1024), "k": log_int(256, 7168), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    elif kind == "linear":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = {"kind": kind, "m": log_int(1, 8192), "n": log_int(64, 4096), "k": log_int(64, 4096), "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"])}
    else:
        c = {"kind": kind, "rows": log_int(1, 2048), "hidden": log_int(256, 8192) // 8 * 8, "n": log_int(256, 8192) // 2 * 2}
    c.pop("name", None)
    return c


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------------------------------- MXFP4 in 32 bits
def _blocks(x):
    """Rows of whole blocks of 32 (zeros behind the last element), in fp32."""
    x = x.float()
    pad = -x.shape[1] % 32
    return (torch.nn.functional.pad(x, (0, pad)) if pad else x).unflatten(1, (-1, 32))


def _power(e):
    """2^e as fp32, -126 <= e <= 127."""
    return ((e + 127) << 23).view(torch.float32)


def _quantized(x):
    """Blocks of 32 and their exponents: E2M1 values v and e with x near v 2^e: y = x / 2^e, the index of its |v|, e."""
    b = _blocks(x)
    bits = (b.abs().amax(2).clamp(min=FLOOR) / 6).view(torch.int32)
    e = ((bits >> 23) + (bits & 0x7FFFFF).ne(0)).clamp(1, 254) - 127
    y = b / _power(e)[:, :, None]
    index = torch.bucketize(y.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device))
    return y, index, e


def _rounded(x):
    """The values that MXFP4 rows of x stand for, in fp32."""
    y, index, e = _quantized(x)
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)[index]
    return (torch.where(y < 0, -v, v) * _power(e)[:, :, None]).flatten(1)


def _packed(x):
    """(codes, scales) of x's rows: two E2M1 codes a byte, the first in the low half, and an E8M0 byte a block."""
    y, index, e = _quantized(x)
    code = (index + 8 * ((y < 0) & (index > 0))).flatten(1).to(torch.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, (e + 127).to(torch.uint8)


def _unpacked(pair):
    codes, scales = pair
    code = torch.stack([codes & 15, codes >> 4], 2).flatten(1).int()
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)[code]
    return (v.unflatten(1, (-1, 32)) * _power(scales.int() - 127)[:, :, None]).flatten(1)


def prepare(case, seed):
    g = _generator(seed)
    randn = lambda shape, scale=1.0, shift=0.0: torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(shift)
    # rows as a block leaves them: some channels are wider than others
    rows = lambda t, h, scale=1.0: randn((t, h), scale).mul_(randn((h,), 0.7).exp_())
    s = {"case": case}
    kind = case["kind"]
    if kind in ("norm", "norm_gemm"):
        T, H = case["rows"], case["hidden"]
        dt, wdt = DT[case.get("dtype", "bf16")], DT[case.get("wdtype", "bf16")]
        s["x"] = rows(T, H).add_(0.3).to(dt)
        s["r"] = rows(T, H, 1.5).add_(0.5).to(dt) if case.get("residual", True) else None
        s["w"] = randn((H,), 0.1, 1.0).to(wdt)
        s["b"] = randn((H,), 0.1).to(wdt) if case.get("bias", True) else None
        if kind == "norm_gemm":
            s["q"] = _packed(randn((case["n"], H), 0.02))
            s["d"] = torch.empty((T, case["n"]), dtype=torch.bfloat16, device="cuda")
        if case.get("train"):
            s["dr"], s["dh"] = randn((T, H), 0.1).to(dt), randn((T, H), 0.1).to(dt)
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["r"], s["w"], s["b"]) if t is not None]
    elif kind == "gemm":
        m, n, k, dt = case["m"], case["n"], case["k"], DT[case["out"]]
        s["a"], s["q"] = _packed(rows(m, k)), _packed(randn((n, k), 0.02))
        s["c"] = {"none": None, "matrix": (m, n), "bias": (n,)}[case["add"]]
        s["c"] = None if s["c"] is None else randn(s["c"]).to(dt)
        s["d"] = torch.empty((m, n // 2 if case["swiglu"] else n), dtype=dt, device="cuda")
    elif kind == "quant_gemm":
        s["x"] = rows(case["m"], case["k"]).to(DT[case["dtype"]])
        s["q"] = _packed(randn((case["n"], case["k"]), 0.02))
        s["d"] = torch.empty((case["m"], case["n"]), dtype=torch.bfloat16, device="cuda")
    else:
        m, n, k, dt = case["m"], case["n"], case["k"], DT[case["dtype"]]
        s["x"] = rows(m, k).to(dt).requires_grad_()
        s["w"] = randn((n, k), 0.02).to(DT[case["wdtype"]]).requires_grad_()
        s["dy"] = randn((m, n), 1e-2).to(dt)
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    c = s["case"]
    dt, scale = s["x"].dtype, c.get("scale", 1.0)
    t = scale * s["x"].float()
    if s["r"] is not None:
        t = s["r"].float() + t
    centred = t - t.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    u = centred * rstd
    h = u * s["w"].float()
    if s["b"] is not None:
        h = h + s["b"].float()
    out = {"residual": t.to(dt), "h": h.to(dt)}
    if not c.get("train"):
        return out
    dh = s["dh"].float()
    du = dh * s["w"].float()
    total = s["dr"].float() + rstd * (du - du.mean(1, keepdim=True) - u * (du * u).mean(1, keepdim=True))
    out["dw"] = (dh * u).double().sum(0).to(s["w"].dtype)
    if s["b"] is not None:
        out["db"] = dh.double().sum(0).to(s["w"].dtype)
    if s["r"] is not None:
        out["dr"] = total.to(dt)
    out["dx"] = (scale * total).to(dt)
    return out


def _plain_gemm(a, b, add=None, swiglu=False, dtype=torch.bfloat16):
    d = a @ b.t()
    if swiglu:
        gate, up = d.chunk(2, dim=1)
        gate = gate.clamp(max=CLAMP)
        d = gate / (1 + torch.exp(-gate)) * up.clamp(-CLAMP, CLAMP)
    elif add is not None:
        d = d + add.float()
    return d.to(dtype)


def _plain_linear(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    return {"y": _plain_gemm(_rounded(x), _rounded(w), dtype=x.dtype),
            "dx": _plain_gemm(_rounded(dy), _rounded(w.t()), dtype=x.dtype),
            "dw": _plain_gemm(_rounded(dy.t()), _rounded(x.t()), dtype=w.dtype)}


# ------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    import hopper_megamoe_basedondeepgemm_amd as moe
    c = s["case"]
    if c["kind"] == "norm":
        r, h = moe.layer_norm_residual(s["x"], s["r"], s["w"], s["b"], residual_scale=c["scale"], eps=EPS)
        out = {"residual": r, "h": h}
        if c["train"]:
            grads = list(torch.autograd.grad((r, h), s["leaves"], (s["dr"], s["dh"])))
            out["dx"] = grads.pop(0)
            if s["r"] is not None:
                out["dr"] = grads.pop(0)
            out["dw"] = grads.pop(0)
            if s["b"] is not None:
                out["db"] = grads.pop(0)
        return out
    if c["kind"] == "norm_gemm":
        r, h, rows = moe.layer_norm_residual(s["x"], s["r"], s["w"], s["b"], eps=EPS, quant="mxfp4")
        moe.mxfp4_gemm_nt(rows, s["q"], s["d"])
        return {"residual": r, "h": h, "d": s["d"]}
    if c["kind"] == "quant_gemm":
        moe.mxfp4_gemm_nt(moe.mxfp4_quantize(s["x"]), s["q"], s["d"])
        return s["d"]
    if c["kind"] == "gemm":
        moe.mxfp4_gemm_nt(s["a"], s["q"], s["d"], c=s["c"], activation="swiglu" if c["swiglu"] else None, activation_clamp=CLAMP)
        return s["d"]
    y = moe.mxfp4_linear(s["x"], s["w"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        s, c = state, state["case"]
        if c["kind"] == "norm":
            return _plain_norm(s)
        if c["kind"] == "norm_gemm":
            out = _plain_norm(s)
            return dict(out, d=_plain_gemm(_rounded(out["h"]), _unpacked(s["q"])))
        if c["kind"] == "quant_gemm":
            return _plain_gemm(_rounded(s["x"]), _unpacked(s["q"]))
        if c["kind"] == "gemm":
            return _plain_gemm(_unpacked(s["a"]), _unpacked(s["q"]), s["c"], c["swiglu"], DT[c["out"]])
        return _plain_linear(s)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    mx = lambda values: values * 17 / 32
    if case["kind"] == "norm":
        T, H, e, w = case["rows"], case["hidden"], size[case["dtype"]], size[case["wdtype"]]
        row, weights = T * H * e, (2 if case["bias"] else 1) * H * w
        b = (4 if case["residual"] else 3) * row + weights
        if case["train"]:
            b += (4 if case["residual"] else 3) * row + weights
        return {"bytes": b, "flops": T * H * (26 if case["train"] else 10)}
    if case["kind"] == "norm_gemm":
        T, H, n = case["rows"], case["hidden"], case["n"]
        return {"bytes": 8 * T * H + 4 * H + mx(n * H) + 2 * T * n, "flops": 2 * T * H * n}
    m, n, k = case["m"], case["n"], case["k"]
    if case["kind"] == "quant_gemm":
        return {"bytes": m * k * size[case["dtype"]] + mx(n * k) + 2 * m * n, "flops": 2 * m * n * k}
    if case["kind"] == "gemm":
        e = size[case["out"]]
        out = m * n * e // (2 if case["swiglu"] else 1)
        return {"bytes": mx((m + n) * k) + out + {"none": 0, "matrix": out, "bias": n * e}[case["add"]], "flops": 2 * m * n * k}
    e, w = size[case["dtype"]], size[case["wdtype"]]
    return {"bytes": 2 * (m * k + m * n) * e + 2 * n * k * w, "flops": 6 * m * n * k}


# ------------------------------------------------------------------------------------------- 64 bits
def _exact_power(e):
    """2^e by its bits (a power function's may miss a tie between two codes)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_values(x):
    """MXFP4's values of x's rows: the least power of two that brings a block within 6, and on each of the three ranges of
    E2M1 the nearest multiple of its step, halves towards zero."""
    t, k = x.double(), x.shape[1]
    t = torch.cat([t, t.new_zeros(t.shape[0], -k % 32)], 1).reshape(t.shape[0], -1, 32)
    mantissa, exponent = torch.frexp(t.abs().amax(2, keepdim=True).clamp(min=FLOOR) / 6)
    unit = _exact_power((exponent - (mantissa == 0.5).int()).clamp(-126, 127))
    a = t.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.ceil(a / step - 0.5) * step).clamp(max=6)
    return (torch.sign(t) * a * unit).flatten(1)


def _exact_codes(pair):
    """The values that (codes, scales) stand for: E2M1 by its sign, exponent and mantissa bits."""
    codes, scales = pair
    c = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.int32, device=codes.device)
    c[:, 0::2], c[:, 1::2] = codes % 16, codes // 16
    e, m = (c // 2 % 4).double(), (c % 2).double()
    v = torch.where(e > 0, (1 + m / 2) * _exact_power(e - 1), m / 2) * (1 - 2 * (c // 8)).double()
    return v * _exact_power(scales.int() - 127).repeat_interleave(32, dim=1)


def _exact_product(a, b):
    return a.mm(b.t().contiguous())


def _exact_norm(s, x, r, w, b):
    total = s["case"].get("scale", 1.0) * x + (0 if r is None else r)
    deviation = total - total.mean(-1, keepdim=True)
    h = deviation / torch.sqrt(deviation.square().mean(-1, keepdim=True) + EPS) * w
    return total, h if b is None else h + b


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "norm_gemm"):
        v = {k: None if s[k] is None else s[k].detach().double() for k in ("x", "r", "w", "b")}
        if case.get("train"):
            on = [k for k in v if v[k] is not None]
            for k in on:
                v[k].requires_grad_()
            r, h = _exact_norm(s, **v)
            grads = torch.autograd.grad((r, h), [v[k] for k in on], (s["dr"].double(), s["dh"].double()))
            return dict({"residual": r.detach(), "h": h.detach()}, **{"d" + k: t for k, t in zip(on, grads)})
        r, h = _exact_norm(s, **v)
        if case["kind"] == "norm":
            return {"residual": r, "h": h}
        return {"residual": r, "h": h, "d": _exact_product(_exact_values(h.to(torch.bfloat16)), _exact_codes(s["q"]))}
    if case["kind"] == "quant_gemm":
        return _exact_product(_exact_values(s["x"]), _exact_codes(s["q"]))
    if case["kind"] == "gemm":
        d = _exact_product(_exact_codes(s["a"]), _exact_codes(s["q"]))
        if case["swiglu"]:
            half = d.shape[1] // 2
            gate = torch.minimum(d[:, :half], d.new_tensor(CLAMP))
            return gate / (1 + torch.exp(-gate)) * d[:, half:].clamp(-CLAMP, CLAMP)
        return d if s["c"] is None else d + s["c"].double()
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
    return {"y": _exact_product(_exact_values(x), _exact_values(w)), "dx": _exact_product(_exact_values(dy), _exact_values(w.t())),
            "dw": _exact_product(_exact_values(dy.t()), _exact_values(x.t()))}
