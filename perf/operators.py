"""The operators around the MoE layer that are timed: one pass of each case through the public entry points.

  norm       the norm behind one block, its gate and residual scale and the norm before the next one
             (``rms_norm_residual``); with "train" the backward pass too
  norm_gemm  the same with int8 rows for the dense expert, and their product with its weights
  gemm       int8 rows times int8 weights (``int8_gemm_nt``): plain, added to C or a bias, or with SwiGLU
  balance    the router's balance loss and per-expert counts, and the gradient of its logits
             (``router_balance_loss``)

With ``own`` false, ``run`` computes the same in elementary torch operations, in 32 bits (column sums over
tokens in 64). ``exact`` restates the operators in 64 bits, gradients by differentiation.
"""
import math

import torch

own = False
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS, CLAMP, ALPHA, BETA = 1e-6, 10.0, 0.01, 0.001


def _norm(name, rows, hidden, dtype="bf16", wdtype="bf16", post=True, gate="none", sigmoid=False, scale=1.0, train=False):
    return {"name": name, "kind": "norm", "rows": rows, "hidden": hidden, "dtype": dtype, "wdtype": wdtype, "post": post,
            "gate": gate, "sigmoid": sigmoid, "scale": scale, "train": train}


def _gemm(name, m, n, k, out="bf16", add="none", swiglu=False):
    return {"name": name, "kind": "gemm", "m": m, "n": n, "k": k, "out": out, "add": add, "swiglu": swiglu}


def _balance(name, tokens, experts, topk, dtype="fp32", score="softmax", seqs=1, padded=0.0):
    return {"name": name, "kind": "balance", "tokens": tokens, "experts": experts, "topk": topk, "dtype": dtype, "score": score,
            "seqs": seqs, "padded": padded}


def listed():
    return [
        # one sequence being decoded: residual add and the norm before the layer
        _norm("norm-m1-h4096", 1, 4096, post=False),
        # a prefill chunk: post norm, channel gate, scaled residual add, next norm
        _norm("norm-m8192-h4096-post-gate", 8192, 4096, gate="channel", scale=0.22),
        # a training step of the same with a sigmoid gate for each token, fp32 norm weights
        _norm("norm-train-m4096-h4096", 4096, 4096, wdtype="fp32", gate="token", sigmoid=True, train=True),
        # a ragged training batch in fp32, a gate for each element
        _norm("norm-train-m777-h2880-fp32", 777, 2880, dtype="fp32", wdtype="fp32", gate="full", scale=0.5, train=True),
        # a decode batch into the dense expert: norm, int8 rows, product
        {"name": "norm-gemm-m64-h7168-n4096", "kind": "norm_gemm", "rows": 64, "hidden": 7168, "n": 4096},
        # single token, down projection of the dense expert added to the experts' output
        _gemm("gemm-m1-n4096-k2048-add", 1, 4096, 2048, add="matrix"),
        # a ragged decode batch, gate and up projection with SwiGLU
        _gemm("gemm-m37-n8192-k4096-swiglu", 37, 8192, 4096, swiglu=True),
        # an odd prefill chunk with a bias, fp16 out
        _gemm("gemm-m1000-n5120-k2880-bias-fp16", 1000, 5120, 2880, out="fp16", add="bias"),
        # the largest: a prefill of 8192 tokens
        _gemm("gemm-m8192-n8192-k4096", 8192, 8192, 4096),
        # a decode batch's counts and loss
        _balance("balance-m64-e384", 64, 384, 8),
        # packed training sequences of uneven lengths, some tokens padded
        _balance("balance-m16384-e384-seqs", 16384, 384, 8, seqs=24, padded=0.05),
        # a large micro-batch with bf16 logits and sigmoid scores
        _balance("balance-m65536-e256-sigmoid", 65536, 256, 8, dtype="bf16", score="sigmoid"),
    ]


def draw(rng):
    log_int = lambda lo, hi: min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))
    kind = rng.choice(["norm", "norm", "gemm", "gemm", "balance", "norm_gemm"])
    if kind == "norm":
        hidden = log_int(256, 8192)
        hidden = hidden if rng.random() < 0.2 else max(8, hidden // 8 * 8)
        rows = log_int(1, max(1, min(8192, 8192 * 4096 // hidden)))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = _norm("", rows, hidden, dtype, rng.choice([dtype, "fp32"]), rng.random() < 0.6, rng.choice(["none", "channel", "token", "full"]),
                  rng.random() < 0.5, rng.choice([1.0, 0.22, 0.5]), rows <= 4096 and rng.random() < 0.5)
    elif kind == "gemm":
        n, k = log_int(256, 8192) // 2 * 2, log_int(256, 8192) // 16 * 16
        m = log_int(1, max(1, min(8192, 8192 * 8192 * 4096 // (n * k))))
        swiglu = rng.random() < 0.3
        c = _gemm("", m, n, k, rng.choice(["bf16", "bf16", "fp16", "fp32"]), "none" if swiglu else rng.choice(["none", "matrix", "bias"]), swiglu)
    elif kind == "balance":
        experts = log_int(8, 512)
        tokens = log_int(1, 65536)
        c = _balance("", tokens, experts, min(experts, rng.choice([1, 2, 4, 8])), rng.choice(["fp32", "bf16"]), rng.choice(["softmax", "sigmoid"]),
                     rng.choice([1, min(tokens, log_int(1, 64))]), rng.choice([0.0, 0.05, 0.5]))
    else:
        c = {"kind": "norm_gemm", "rows": log_int(1, 2048), "hidden": log_int(256, 8192) // 16 * 16, "n": log_int(256, 8192) // 2 * 2}
    c.pop("name", None)
    return c


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int8(g, rows, k):
    """Rows as a cast leaves them: integers of a bell shape up to 127 and a scale for each row."""
    q = torch.randn((rows, k), generator=g, device="cuda").mul_(33.0).round_().clamp_(-127, 127).to(torch.int8)
    return q, torch.rand((rows,), generator=g, device="cuda").mul_(0.02).add_(0.01)


def prepare(case, seed):
    g = _generator(seed)
    randn = lambda shape, scale=1.0, shift=0.0: torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(shift)
    s = {"case": case}
    kind = case["kind"]
    if kind in ("norm", "norm_gemm"):
        T, H = case["rows"], case["hidden"]
        dt, wdt = DT[case.get("dtype", "bf16")], DT[case.get("wdtype", "bf16")]
        s["x"], s["r"] = randn((T, H), 0.7).to(dt), randn((T, H), 1.5).to(dt)
        s["post"] = randn((H,), 0.1, 1.0).to(wdt) if case.get("post") else None
        s["pre"] = randn((H,), 0.1, 1.0).to(wdt)
        shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[case.get("gate", "none")]
        s["gate"] = None if shape is None else randn(shape, 0.5, 0.5).to(dt)
        if kind == "norm_gemm":
            s["b"] = _int8(g, case["n"], H)
            s["d"] = torch.empty((T, case["n"]), dtype=torch.bfloat16, device="cuda")
        if case.get("train"):
            s["dr"], s["dh"] = randn((T, H), 0.1).to(dt), randn((T, H), 0.1).to(dt)
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["r"], s["post"], s["pre"], s["gate"]) if t is not None]
    elif kind == "gemm":
        m, n, k, dt = case["m"], case["n"], case["k"], DT[case["out"]]
        s["a"], s["b"] = _int8(g, m, k), _int8(g, n, k)
        s["c"] = {"none": None, "matrix": (m, n), "bias": (n,)}[case["add"]]
        s["c"] = None if s["c"] is None else randn(s["c"], 10.0).to(dt)
        s["d"] = torch.empty((m, n // 2 if case["swiglu"] else n), dtype=dt, device="cuda")
    else:
        T, E, B = case["tokens"], case["experts"], case["seqs"]
        s["logits"] = (randn((T, E)) + randn((E,), 0.5)).to(DT[case["dtype"]])
        s["idx"] = s["logits"].float().topk(case["topk"], dim=1).indices
        s["idx"][torch.rand((T,), generator=g, device="cuda") < case["padded"]] = -1
        s["logits"].requires_grad_()
        cuts = torch.rand((B - 1,), generator=g, device="cuda").mul_(T + 1).long().clamp_(max=T).sort().values
        s["cu"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), T)]).int() if B > 1 else None
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    c = s["case"]
    x, r = s["x"].float(), s["r"].float()
    scale = c.get("scale", 1.0)
    a = None if s["gate"] is None else (torch.sigmoid(s["gate"].float()) if c["sigmoid"] else s["gate"].float())
    n = x
    if s["post"] is not None:
        rstd1 = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
        z = x * rstd1
        n = z * s["post"].float()
    t = r + scale * (n if a is None else a * n)
    rstd2 = torch.rsqrt((t * t).mean(1, keepdim=True) + EPS)
    u = t * rstd2
    h = u * s["pre"].float()
    dt = s["x"].dtype
    out = {"residual": t.to(dt), "h": h.to(dt)}
    if not c.get("train"):
        return out
    dh = s["dh"].float()
    du = dh * s["pre"].float()
    dt_ = s["dr"].float() + rstd2 * (du - u * (du * u).mean(1, keepdim=True))
    out["dpre"] = (dh * u).sum(0).to(s["pre"].dtype)
    out["dr"] = dt_.to(dt)
    dn = scale * dt_
    if a is not None:
        da = dn * n
        dn = dn * a
        if c["gate"] == "token":
            da = da.sum(1, keepdim=True)
        elif c["gate"] == "channel":
            da = da.sum(0)
        out["dgate"] = (da * a * (1 - a) if c["sigmoid"] else da).to(dt)
    if s["post"] is not None:
        out["dpost"] = (dn * z).sum(0).to(s["post"].dtype)
        dz = dn * s["post"].float()
        dn = rstd1 * (dz - z * (dz * z).mean(1, keepdim=True))
    out["dx"] = dn.to(dt)
    return out


def _plain_gemm(a, b, add=None, swiglu=False, dtype=torch.bfloat16):
    d = (a[0].float() @ b[0].float().t()) * (a[1][:, None] * b[1])
    if swiglu:
        gate, up = d.chunk(2, dim=1)
        d = torch.nn.functional.silu(gate.clamp(max=CLAMP)) * up.clamp(-CLAMP, CLAMP)
    elif add is not None:
        d = d + add.float()
    return d.to(dtype)


def _plain_norm_gemm(s):
    out = _plain_norm(s)
    h = out["h"].float()
    sf = h.abs().amax(1).clamp(min=1e-30) / 127.0
    q = torch.round(h / sf[:, None]).clamp(-127, 127)
    out["d"] = _plain_gemm((q, sf), s["b"])
    return out


def _plain_balance(s):
    c = s["case"]
    logits, idx = s["logits"].float(), s["idx"]
    T, E, B = c["tokens"], c["experts"], c["seqs"]
    seq = torch.zeros(T, dtype=torch.long, device=idx.device)
    if s["cu"] is not None:
        seq = torch.searchsorted(s["cu"][1:].long(), torch.arange(T, device=idx.device), right=True)
    slots = idx >= 0
    routed = slots.any(1)
    counts = torch.zeros(B * E + 1, dtype=torch.long, device=idx.device)
    counts.scatter_add_(0, torch.where(slots, seq[:, None] * E + idx, B * E).flatten(), torch.ones_like(idx).flatten())
    counts = counts[:-1].view(B, E)
    lse = torch.logsumexp(logits, dim=1)
    if c["score"] == "softmax":
        p, z = torch.softmax(logits, dim=1), BETA
    else:
        sig = torch.sigmoid(logits)
        p, z = sig / sig.sum(1, keepdim=True), 0.0
    member = ((seq[:, None] == torch.arange(B, device=idx.device)) & routed[:, None]).double()
    n = member.sum(0)
    f = E * counts.double() / counts.sum(1, keepdim=True).clamp(min=1)
    P = (member.t() @ p.double()) / n.clamp(min=1)[:, None]
    live, total = (n > 0).sum().clamp(min=1), n.sum().clamp(min=1)
    loss = ALPHA / live * (f * P).sum() + z / total * (lse.double() ** 2 * routed).sum()
    coef = (ALPHA / (live * n.clamp(min=1))).float()[seq] * routed
    ft = f.float()[seq]
    grad = coef[:, None] * p * (ft - (ft * p).sum(1, keepdim=True))
    grad = grad * (1 - sig) if c["score"] == "sigmoid" else grad + (2 * z / total.float() * lse * routed)[:, None] * p
    return {"loss": loss.float(), "counts": (counts if B > 1 else counts[0]).int(), "dlogits": grad.to(s["logits"].dtype)}


# ------------------------------------------------------------------------------------------- the framework's calls
def _own_norm(moe, s):
    c = s["case"]
    r, h = moe.rms_norm_residual(s["x"], s["r"], post_weight=s["post"], gate=s["gate"], gate_sigmoid=c["sigmoid"],
                                 residual_scale=c["scale"], pre_weight=s["pre"], eps=EPS)
    out = {"residual": r, "h": h}
    if c["train"]:
        grads = list(torch.autograd.grad((r, h), s["leaves"], (s["dr"], s["dh"])))
        out["dpre"] = grads[3 if s["post"] is not None else 2]
        out["dr"] = grads[1]
        if s["gate"] is not None:
            out["dgate"] = grads[-1]
        if s["post"] is not None:
            out["dpost"] = grads[2]
        out["dx"] = grads[0]
    return out


def _own(s):
    import hopper_megamoe_basedondeepgemm_amd as moe
    c = s["case"]
    if c["kind"] == "norm":
        return _own_norm(moe, s)
    if c["kind"] == "norm_gemm":
        r, h, rows = moe.rms_norm_residual(s["x"], s["r"], pre_weight=s["pre"], eps=EPS, quant="int8")
        moe.int8_gemm_nt(rows, s["b"], s["d"])
        return {"residual": r, "h": h, "d": s["d"]}
    if c["kind"] == "gemm":
        moe.int8_gemm_nt(s["a"], s["b"], s["d"], c=s["c"], activation="swiglu" if c["swiglu"] else None, activation_clamp=CLAMP)
        return s["d"]
    loss, counts = moe.router_balance_loss(s["logits"], s["idx"], cu_seqlens=s["cu"], balance_coef=ALPHA, score=c["score"],
                                           z_coef=BETA if c["score"] == "softmax" else 0.0)
    return {"loss": loss.detach(), "counts": counts, "dlogits": torch.autograd.grad(loss, s["logits"])[0]}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        c = state["case"]
        if c["kind"] == "norm":
            return _plain_norm(state)
        if c["kind"] == "norm_gemm":
            return _plain_norm_gemm(state)
        if c["kind"] == "gemm":
            return _plain_gemm(state["a"], state["b"], state["c"], c["swiglu"], DT[c["out"]])
        return _plain_balance(state)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["kind"] == "norm":
        T, H, e = case["rows"], case["hidden"], size[case["dtype"]]
        full = T * H * e if case["gate"] == "full" else 0
        b = 4 * T * H * e + full + 2 * H * size[case["wdtype"]]
        if case["train"]:
            b += 6 * T * H * e + 2 * full + 4 * H * size[case["wdtype"]]
        return {"bytes": b, "flops": T * H * (40 if case["train"] else 12)}
    if case["kind"] == "norm_gemm":
        T, H, n = case["rows"], case["hidden"], case["n"]
        return {"bytes": 8 * T * H + n * H + 2 * T * n + 4 * (T + n), "flops": 2 * T * H * n}
    if case["kind"] == "gemm":
        m, n, k, e = case["m"], case["n"], case["k"], size[case["out"]]
        out = m * n * e // (2 if case["swiglu"] else 1)
        return {"bytes": m * k + n * k + 4 * (m + n) + out + {"none": 0, "matrix": out, "bias": n * e}[case["add"]], "flops": 2 * m * n * k}
    T, E = case["tokens"], case["experts"]
    return {"bytes": 3 * T * E * size[case["dtype"]] + 8 * T * case["topk"] + 4 * E * case["seqs"], "flops": 16 * T * E}


# ------------------------------------------------------------------------------------------- 64 bits
def _exact_norm(s, x, r, post, pre, gate):
    c = s["case"]
    rms = lambda v: v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
    n = x if post is None else rms(x) * post
    if gate is not None:
        n = n * (1 / (1 + torch.exp(-gate)) if c["sigmoid"] else gate)
    total = r + c.get("scale", 1.0) * n
    return total, rms(total) * pre


def _exact_gemm(a, b):
    return a[0].double().mm(b[0].double().t().contiguous()) * a[1].double()[:, None] * b[1].double()[None, :]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "norm_gemm"):
        names = ["x", "r", "post", "pre", "gate"]
        v = {k: None if s[k] is None else s[k].detach().double() for k in names}
        if case.get("train"):
            on = [k for k in names if v[k] is not None]
            for k in on:
                v[k].requires_grad_()
            r, h = _exact_norm(s, **v)
            grads = dict(zip(on, torch.autograd.grad((r, h), [v[k] for k in on], (s["dr"].double(), s["dh"].double()))))
            out = {"residual": r.detach(), "h": h.detach(), "dpre": grads["pre"], "dr": grads["r"]}
            if s["gate"] is not None:
                out["dgate"] = grads["gate"]
            if s["post"] is not None:
                out["dpost"] = grads["post"]
            return dict(out, dx=grads["x"])
        r, h = _exact_norm(s, **v)
        if case["kind"] == "norm":
            return {"residual": r, "h": h}
        rows = h.to(torch.bfloat16).double()
        sf = rows.abs().amax(1).clamp(min=1e-30) / 127
        return {"residual": r, "h": h, "d": _exact_gemm(((rows / sf[:, None]).round().clamp(-127, 127), sf), s["b"])}
    if case["kind"] == "gemm":
        d = _exact_gemm(s["a"], s["b"])
        if case["swiglu"]:
            half = d.shape[1] // 2
            gate = torch.minimum(d[:, :half], d.new_tensor(CLAMP))
            return gate / (1 + torch.exp(-gate)) * d[:, half:].clamp(-CLAMP, CLAMP)
        return d if s["c"] is None else d + s["c"].double()
    T, E, B = case["tokens"], case["experts"], case["seqs"]
    logits = s["logits"].detach().double().requires_grad_()
    cuts = [0, T] if s["cu"] is None else s["cu"].tolist()
    weight = logits.exp() if case["score"] == "softmax" else 1 / (1 + torch.exp(-logits))
    p = weight / weight.sum(1, keepdim=True)
    routed = (s["idx"] >= 0).any(1)
    counts = torch.zeros((B, E), dtype=torch.int32, device=logits.device)
    terms = []
    for i, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])):
        rows = routed[lo:hi]
        hits = s["idx"][lo:hi].flatten()
        counts[i] = torch.bincount(hits[hits >= 0], minlength=E)
        if bool(rows.any()):
            f = counts[i].double() * E / counts[i].sum()
            terms.append((p[lo:hi][rows].mean(0) * f).sum())
    loss = ALPHA * torch.stack(terms).mean() if terms else (logits * 0).sum()
    if case["score"] == "softmax" and terms:
        loss = loss + BETA * torch.log(weight.sum(1))[routed].square().mean()
    return {"loss": loss.detach(), "counts": counts if B > 1 else counts[0], "dlogits": torch.autograd.grad(loss, logits)[0]}
