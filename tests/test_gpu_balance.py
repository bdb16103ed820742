"""router_balance_loss, its counts and gradient against the formula in 64 bits.

Tolerances: a probability is within 2^-24 times (3 + |l - max| for the rounded difference's exponential, 2
units for expf, 22 additions of the sum, 2 for the quotient), below 30 + |l - max|; where |l - max| > 104 the
exponential is below the least fp32 number and may be zero, an absolute error of 2^-126 over the sum (>= 1).
Sums over a chunk's tokens (at most 128 per wave and 4 waves here) add 132, later sums are 64-bit: 256
covers P. The logits here lie within 40 of their maximum (or are -inf). loss: sums of non-negative terms,
so 2^-24 (256 + 40 for lse^2 relative) times itself. Gradient: C 2^-24 times the same formula over absolute
values, with C = 2 (30 + 40) + 24 for the dot = 170, and half a step of its type."""
import pytest
import torch

from tests.gpu_common import need_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(T, E, k, dtype=torch.float32, seed=0, padded=0.2, i64=True):
    torch.manual_seed(seed)
    logits = ((torch.randn((T, E), device="cuda") + torch.randn(E, device="cuda")) * 2).to(dtype)
    idx = torch.argsort(torch.rand((T, E), device="cuda"), dim=1)[:, :k].contiguous()
    idx[torch.rand(T, device="cuda") < padded] = -1
    if k > 1:
        idx[torch.rand(T, device="cuda") < 0.1, -1] = -1          # some slots alone
    return logits, idx if i64 else idx.int()


def formula(logits, idx, cuts, alpha, beta, score):
    """(loss, counts [B, E], gradient for d_loss = 1, the gradient's magnitude), 64 bits, on the CPU"""
    l, idx = logits.detach().double().cpu(), idx.long().cpu()
    T, E = l.shape
    B = len(cuts) - 1
    counts = torch.zeros((B, E), dtype=torch.int64)
    ok = (idx >= 0) & (idx < E)
    routed = ok.any(1)
    alive = torch.isfinite(l).any(1)
    if score == "softmax":
        lse = torch.logsumexp(l, 1)
        p = torch.where(alive[:, None], torch.exp(l - lse[:, None]), torch.zeros_like(l))
        lse = torch.where(alive, lse, torch.zeros_like(lse))
    else:
        sg = torch.sigmoid(l)
        p = torch.where(alive[:, None], sg / sg.sum(1, keepdim=True), torch.zeros_like(l))
        lse = torch.zeros(T, dtype=torch.float64)
    rows = [r for lo, hi in zip(cuts[:-1], cuts[1:]) for r in range(lo, hi) if routed[r]]
    live = 0
    parts = []
    for b, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])):
        h = idx[lo:hi][ok[lo:hi]]
        counts[b] = torch.bincount(h, minlength=E)
        n = int(routed[lo:hi].sum())
        parts.append(n)
        live += n > 0
    N = len(rows)
    loss = 0.0
    grad, mag = torch.zeros_like(l), torch.zeros_like(l)
    for b, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])):
        n = parts[b]
        if n == 0:
            continue
        f = E * counts[b].double() / counts[b].sum()
        on = routed[lo:hi]
        loss += alpha / live * float((f * p[lo:hi][on].mean(0)).sum())
        dot = (p[lo:hi] * f).sum(1, keepdim=True)
        c = alpha / (live * n)
        g, m = c * p[lo:hi] * (f - dot), c * p[lo:hi] * (f + dot)
        if score == "sigmoid":
            g, m = g * (1 - sg[lo:hi]), m
        else:
            z = 2 * beta / N * lse[lo:hi, None] * p[lo:hi]
            g, m = g + z, m + z.abs()
        grad[lo:hi], mag[lo:hi] = g * on[:, None], m * on[:, None]
    if N and score == "softmax":
        loss += beta / N * float(lse[rows].square().sum())
    return loss, counts, grad, mag


def close(got, ref, mag, c=170):
    fi = torch.finfo(got.dtype)
    got = got.detach().double().cpu()
    # (gradients below the least normal number of the type round to its fixed step)
    tol = ref.abs() * (fi.eps / 2) + c * U * mag * (1 + fi.eps) + fi.tiny * fi.eps + 2.0 ** -126
    assert bool(((got - ref).abs() <= tol).all()), float(((got - ref).abs() / tol).max())


def run(logits, idx, cuts, alpha, beta, score, g=1.0, cu=True):
    import hopper_megamoe_basedondeepgemm_amd as dgm
    leaf = logits.detach().requires_grad_()
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda") if cu else None
    loss, counts = dgm.router_balance_loss(leaf, idx, cu, alpha, beta, score)
    (d,) = torch.autograd.grad(loss * g, leaf)
    return loss, counts, d


def check(logits, idx, cuts, alpha, beta, score, cu=True, g=1.0):
    loss, counts, d = run(logits, idx, cuts, alpha, beta, score, g, cu)
    want, wc, wg, wm = formula(logits, idx, cuts, alpha, beta, score)
    assert torch.equal(counts.long().cpu().view(wc.shape), wc) and counts.dtype == torch.int32
    assert loss.dtype == torch.float32 and abs(float(loss.detach()) - want) <= 300 * U * abs(want) + 1e-38
    assert d.dtype == logits.dtype
    close(d, wg * g, wm * abs(g))
    return loss, counts, d


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (2, 64, 64), (5, 65, 3), (64, 384, 8), (100, 128, 2), (256, 512, 8), (257, 100, 4),
                                   (300, 1024, 16), (700, 129, 8), (2000, 256, 8), (9001, 40, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_sequence(T, E, k, dtype):
    need_gpu()
    logits, idx = make(T, E, k, dtype, seed=T + E, i64=T % 2 == 0)
    for score, beta in (("softmax", 0.0), ("softmax", 0.01), ("sigmoid", 0.0)):
        check(logits, idx, [0, T], 0.5, beta, score, cu=False, g=-3.0)


@pytest.mark.parametrize("T,cuts", [(1, [0, 1]), (1, [0, 0, 1, 1]), (40, [0, 1, 2, 3, 3, 3, 17, 40]), (300, [0, 300]), (300, [0, 16, 32, 48, 300]),
                                    (300, [0, 5, 280]), (500, [7, 100, 100, 500]), (64, list(range(65))), (3000, [0, 2999, 3000]),
                                    (3000, [0] * 20 + [1500] * 20 + [3000] * 5), (20000, [0, 3, 9000, 9001, 19990])])
def test_sequences(T, cuts):
    """Lengths of zero and one, sequences that share a chunk, tokens before the first and behind the last."""
    need_gpu()
    logits, idx = make(T, 48, 4, seed=T)
    for score, beta in (("softmax", 0.02), ("sigmoid", 0.0)):
        _, _, d = check(logits, idx, cuts, 1.0, beta, score)
        assert not bool(d[cuts[-1]:].any()) and not bool(d[:cuts[0]].any())


def test_no_tokens_and_nothing_routed():
    need_gpu()
    for T, cuts in ((0, [0, 0]), (0, [0, 0, 0]), (30, [0, 30]), (600, [0, 600]), (600, [0, 100, 600])):
        logits, idx = make(T, 24, 2, seed=1)
        idx[:] = -1
        logits[:] = float("nan")                     # unrouted tokens' logits are not looked at
        loss, counts, d = run(logits, idx, cuts, 1.0, 0.1, "softmax")
        assert float(loss.detach()) == 0.0 and not bool(counts.any()) and not bool(d.any()) and d.shape == logits.shape


def test_masked_experts_and_bad_ids():
    """-inf and the type's lowest value in masked experts, rows of nothing else, ids out of range, NaN in
    unrouted rows, the same id twice."""
    need_gpu()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits, idx = make(400, 96, 4, dtype, seed=3)
        logits[:, 50:] = float("-inf")
        logits[7, :] = float("-inf")
        idx[7] = torch.arange(4, device="cuda")
        idx[8, 0], idx[9, 1], idx[10, 2] = 96, -7, 2 ** 40
        idx[11] = 5
        off = ~((idx >= 0) & (idx < 96)).any(1)
        logits[off] = float("nan")
        clean = logits.clone()
        clean[off] = 0
        for score, beta in (("softmax", 0.01), ("sigmoid", 0.0)):
            loss, counts, d = run(logits, idx, [0, 400], 1.0, beta, score)
            want, wc, wg, wm = formula(clean, idx, [0, 400], 1.0, beta, score)
            assert torch.equal(counts.long().cpu(), wc) and abs(float(loss.detach()) - want) <= 300 * U * abs(want)
            close(d, wg, wm)
            assert not bool(d[off].any()) and not bool(d[7].any()) and not bool(d[:, 50:].any())
        low = logits.masked_fill(torch.isinf(logits), torch.finfo(dtype).min)
        low[7, 0] = 0
        low[off] = 0
        check(low, idx, [0, 400], 1.0, 0.01, "softmax")


def test_offsets_beyond_32_bits_and_refusals():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    logits, idx = make(5, 64, 4, seed=2)
    want = run(logits, idx, [0, 5], 1.0, 0.01, "softmax")
    gap = (1 << 30) + 16
    far = torch.empty(gap * 4 + 64, device="cuda").as_strided((5, 64), (gap, 1)).copy_(logits)
    got = run(far, idx, [0, 5], 1.0, 0.01, "softmax")
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    leaf = logits.clone().requires_grad_()
    loss, counts = dgm.router_balance_loss(leaf, idx)
    assert not counts.requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cpu"):
        dgm.router_balance_loss(logits, idx.cpu())
    with pytest.raises(TypeError, match="stats of"):
        dgm.router_balance_loss_backward(torch.ones((), device="cuda"), logits, idx, counts, counts)


def test_gradient_against_differences():
    need_gpu()
    logits, idx = make(60, 32, 4, seed=8)
    cuts = [0, 20, 21, 60]
    for score, beta in (("softmax", 0.05), ("sigmoid", 0.0)):
        _, _, d = run(logits, idx, cuts, 1.0, beta, score)
        for trial in range(4):
            way = torch.randn((60, 32), dtype=torch.float64)
            e = 1e-5
            base = logits.double().cpu()
            up, dn = (formula(base + s * e * way, idx, cuts, 1.0, beta, score)[0] for s in (1, -1))
            diff = (up - dn) / (2 * e)
            got = float((d.double().cpu() * way).sum())
            # (the difference quotient: e^2 of third derivatives and 64-bit cancellation, below 1e-9)
            assert abs(diff - got) <= 200 * U * float((d.double().cpu() * way).abs().sum()) + 1e-9


def test_strides_frontend_buffer_and_streams():
    """Views with row strides, transposed logits, the frontend's own buffer; same bits on another stream, in
    two calls at once and from a captured pair replayed between eager calls."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    logits, idx = make(500, 96, 4, seed=5)
    want = check(logits, idx, [0, 100, 500], 1.0, 0.01, "softmax")
    wide_l = torch.full((500, 130), 9.0, device="cuda")[:, 17:113].copy_(logits)
    wide_i = torch.full((500, 9), 3, device="cuda")[:, 2:6].copy_(idx)
    for l, i in ((wide_l, wide_i), (logits.t().contiguous().t(), idx.t().contiguous().t())):
        got = run(l, i, [0, 100, 500], 1.0, 0.01, "softmax")
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    torch.manual_seed(0)
    b = dgm.get_fused_symm_buffer_for_mega_moe(None, 16, 40, 4, 512, 256)
    x, rw = torch.randn((33, 512), device="cuda").bfloat16(), torch.randn((16, 512), device="cuda").bfloat16() * 0.05
    x[3] = 0                                                  # (left unrouted by the frontend)
    dgm.fable_router_quant_topk_frontend(x, rw, b)
    _, counts, _ = check(b.logits[:33], b.topk_idx[:33], [0, 33], 1.0, 0.01, "softmax", cu=False)
    assert int(counts.sum()) == 32 * 4
    cu = torch.tensor([0, 100, 500], dtype=torch.int32, device="cuda")

    def both():
        loss, counts, stats = dgm.router_balance_loss_forward(logits, idx, cu, 1.0, 0.01)
        one = torch.ones((), device="cuda")
        return loss, counts, dgm.router_balance_loss_backward(one, logits, idx, counts, stats, cu, 1.0, 0.01)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    here = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) and torch.equal(b_, c) for a, b_, c in zip(here, other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
        with pytest.raises(RuntimeError, match="no autograd under graph capture"):
            dgm.router_balance_loss(logits.detach().requires_grad_(), idx)
    for i in range(3):
        logits.copy_(torch.randn_like(logits))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, both())), i


@pytest.mark.parametrize("way", ["offload", "recompute"])
def test_saved_tensors_that_hooks_bring_back(way):
    """Tensors saved for the backward pass that come back in other memory and strides: the same gradient, bit for bit."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    from torch.utils.checkpoint import checkpoint
    logits, idx = make(300, 64, 4, seed=6)
    cu = torch.tensor([0, 100, 290], dtype=torch.int32, device="cuda")

    def grad(how):
        leaf = logits.t().contiguous().requires_grad_()

        def run(v):
            return dgm.router_balance_loss(v.t(), idx, cu, 1.0, 0.01)[0]
        if how == "offload":
            with torch.autograd.graph.save_on_cpu():
                loss = run(leaf)
        else:
            loss = checkpoint(run, leaf, use_reentrant=False) if how == "recompute" else run(leaf)
        keep = [torch.full((12,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]      # (over given up memory)
        out = torch.autograd.grad(loss, leaf)[0]
        del keep
        return out
    assert torch.equal(grad("plain"), grad(way))


def test_saved_tensors_that_come_back_strided_or_elsewhere():
    """Counts in other strides are read as such; tensors left on the CPU are refused, not read."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    logits, idx = make(300, 64, 4, seed=7)
    cu = torch.tensor([0, 100, 290], dtype=torch.int32, device="cuda")

    def grad(unpack):
        leaf = logits.clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            loss = dgm.router_balance_loss(leaf, idx, cu, 1.0, 0.01)[0]
        return torch.autograd.grad(loss, leaf)[0]
    want = grad(lambda t: t)
    assert torch.equal(want, grad(lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone()))
    for part in ((300, 64), (300, 4), (3,), (2, 64), (12,)):
        with pytest.raises(RuntimeError, match="cpu|GPU"):
            grad(lambda t: t.cpu() if t.shape == part else t)


@pytest.mark.parametrize("turned", [False, True])
def test_several_backward_passes_and_moved_memory(turned):
    """The same graph run twice with other incoming gradients, two graphs alive at once, inputs that are read as copies
    and inputs whose memory is replaced between the passes: the plain call's gradient each time."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    logits, idx = make(700, 96, 4, torch.bfloat16, seed=12)
    cu = torch.tensor([0, 100, 101, 650], dtype=torch.int32, device="cuda")
    every = torch.stack([cu, cu + 7], 1)[:, 0]                   # (strided: read as a copy)
    turn = lambda t: t.t().contiguous().t() if turned else t.clone()
    want = run(logits, idx, cu.tolist(), 1.0, 0.01, "softmax")[2]
    twice = run(logits, idx, cu.tolist(), 1.0, 0.01, "softmax", g=-2.0)[2]
    a, b = turn(logits).requires_grad_(), turn(logits + 1).requires_grad_()
    la, _ = dgm.router_balance_loss(a, turn(idx), every, 1.0, 0.01)
    lb, _ = dgm.router_balance_loss(b, turn(idx), every, 1.0, 0.01)
    keep = [torch.full((700 * 96,), 7, dtype=torch.int32, device="cuda") for _ in range(8)]      # (over given up memory)
    other = torch.autograd.grad(lb, b)[0]
    assert torch.equal(torch.autograd.grad(la * -2.0, a, retain_graph=True)[0], twice)
    assert torch.equal(torch.autograd.grad(la, a, retain_graph=True)[0], want)
    a.data = a.data.clone()
    assert torch.equal(torch.autograd.grad(la, a)[0], want)
    assert torch.equal(other, run(logits + 1, idx, cu.tolist(), 1.0, 0.01, "softmax")[2])
    del keep
