"""layer_norm_residual and its gradients against the formulas in 64 bits.

Tolerances: every element may be off by half a step of its type (finfo.eps / 2 of the value) for the last rounding, and
by C 2^-24 of the same formula over absolute values for the fp32 arithmetic. C counts roundings: a mean over H terms
adds at most 16 per thread, 4 by lane exchange, 3 wave parts and 15 wave sums (< 40); the mean and the variance are two
such sums one behind the other, with the products around them every value is within 128. A gradient holds two more such
means and the recomputed row: 384. A sum over T rows adds at most T more."""
import pytest
import torch

from tests.gpu_common import need_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5
DT = (torch.bfloat16, torch.float16, torch.float32)


def close(got, ref, mag, c):
    """|got - ref| <= half a step of got's type + c 2^-24 mag (and the least normal number)"""
    fi = torch.finfo(got.dtype)
    tol = ref.abs() * (fi.eps / 2) + c * U * mag * (1 + fi.eps) + fi.tiny
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((off / tol).max()), got.dtype)


class Form:
    """The formulas in 64 bits, and the same over absolute values (for the error of fp32 sums)."""

    def __init__(self, x, r, w, b, s, eps=EPS):
        d = lambda t: None if t is None else t.detach().double()
        x, r, w, b = d(x), d(r), d(w), d(b)
        self.s = s
        self.t = s * x + (0 if r is None else r)
        self.t_mag = abs(s) * x.abs() + (0 if r is None else r.abs())
        dev = self.t - self.t.mean(1, keepdim=True)
        dev_mag = self.t_mag + self.t_mag.mean(1, keepdim=True)
        self.rstd = torch.rsqrt(dev.square().mean(1, keepdim=True) + eps)
        self.u = dev * self.rstd
        z_mag = dev_mag * self.rstd
        # (the mean of dev^2 takes dev's absolute error, 2 dev d(dev), halved by the root)
        self.u_mag = z_mag + self.u.abs() * ((self.u.abs() * z_mag).mean(1, keepdim=True) + 1)
        self.w = torch.ones_like(self.u[0]) if w is None else w
        self.h = self.u * self.w + (0 if b is None else b)
        self.h_mag = self.u_mag * self.w.abs() + (0 if b is None else b.abs())

    def grads(self, dr, dh):
        """{name: (value, magnitude)}"""
        out = {}
        R = torch.zeros_like(self.t) if dr is None else dr.double()
        Rm = R.abs()
        if dh is not None:
            D = dh.double()
            du = D * self.w
            mean, m = du.mean(1, keepdim=True), (du * self.u).mean(1, keepdim=True)
            mean_mag, mm = du.abs().mean(1, keepdim=True), (du.abs() * self.u_mag).mean(1, keepdim=True)
            out["weight"] = ((D * self.u).sum(0), (D.abs() * self.u_mag).sum(0))
            out["bias"] = (D.sum(0), D.abs().sum(0))
            spread = (self.u.abs() * self.u_mag).mean(1, keepdim=True) + 1          # rstd's own error
            Rm = Rm + self.rstd * (du.abs() + mean_mag + self.u_mag * m.abs() + self.u_mag * mm) * spread
            R = R + self.rstd * (du - mean - self.u * m)
        out["residual"] = (R, Rm)
        out["x"] = (self.s * R, abs(self.s) * Rm)
        return out


def make(T, H, dtype, wdtype, residual=True, weight=True, bias=True, seed=0, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    x = (rnd(T, H) + shift).to(dtype)
    r = (rnd(T, H) * 1.5 - shift / 2).to(dtype) if residual else None
    w = (1 + 0.2 * rnd(H)).to(wdtype) if weight else None
    b = (0.3 * rnd(H)).to(wdtype) if bias else None
    return x, r, w, b, rnd(T, H).to(dtype), rnd(T, H).to(dtype)


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 100), (4, 512), (3, 513), (9, 1024), (2, 1032), (7, 2880), (2, 4096), (1, 4104),
          (3, 8192), (2, 8200), (2, 12345), (1, 16384), (300, 512), (257, 1000), (300, 2048), (258, 2880), (260, 7168), (257, 9000), (300, 33),
          (4200, 64)]
PARTS = [(True, True, True, 1.0, None), (True, True, False, 0.22, torch.float32), (False, True, True, 1.0, torch.float32),
         (False, False, False, -2.0, None), (True, False, True, 0.5, None), (False, True, False, 1.0, None)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype", DT)
def test_forward_and_backward(T, H, dtype):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for residual, weight, bias, s, wdt in PARTS:
        x, r, w, b, dr, dh = make(T, H, dtype, wdt or dtype, residual, weight, bias, seed=T * H)
        f = Form(x, r, w, b, s)
        got_r, got_h = dgm.layer_norm_residual(x, r, w, b, residual_scale=s)
        if r is None and s == 1.0:
            assert got_r is x
        else:
            close(got_r, f.t, f.t_mag, 128)
        close(got_h, f.h, f.h_mag, 128)
        r2, h2, mean, rstd = dgm.layer_norm_residual_forward(x, r, w, b, residual_scale=s)
        assert torch.equal(r2, got_r) and torch.equal(h2, got_h) and mean.shape == rstd.shape == (T,)
        for gr, gh in ((dr, dh), (None, dh), (dr, None)):
            got = dgm.layer_norm_residual_backward(gr, gh, x, r, mean, rstd, w, b, residual_scale=s)
            want = f.grads(gr, gh)
            for name, t, given in zip(("x", "residual", "weight", "bias"), got, (x, r, w, b)):
                assert (t is None) == (given is None)
                if t is not None:
                    value, mag = want.get(name, (torch.zeros(H, device="cuda", dtype=torch.float64),) * 2)
                    close(t, value, mag, 384 + (T if name in ("weight", "bias") else 0))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,H", [(5, 96), (300, 1000), (70, 4096)])
def test_autograd(T, H, dtype):
    """The same through autograd, every set of leaves; r's gradient meets h's where r is x itself."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for residual, weight, bias, s, wdt in PARTS:
        x, r, w, b, dr, dh = make(T, H, dtype, wdt or dtype, residual, weight, bias, seed=T + H)
        want = dgm.layer_norm_residual_backward(dr, dh, x, r, *dgm.layer_norm_residual_forward(x, r, w, b, s)[2:], w, b, s)
        named = [(t, g) for t, g in zip((x, r, w, b), want) if t is not None]
        for t, _ in named:
            t.requires_grad_()
        out = dgm.layer_norm_residual(x, r, w, b, residual_scale=s)
        got = torch.autograd.grad(out, [t for t, _ in named], (dr, dh))
        assert all(torch.equal(a, g) for a, (_, g) in zip(got, named))
        for t, g in named:                   # one leaf at a time, gradients of h alone
            alone = dgm.layer_norm_residual_backward(None, dh, x, r, *dgm.layer_norm_residual_forward(x, r, w, b, s)[2:], w, b, s)
            leaves = [u.detach().requires_grad_(u is t) if u is not None else None for u in (x, r, w, b)]
            out = dgm.layer_norm_residual(*leaves, residual_scale=s)
            i = [u is t for u in (x, r, w, b)].index(True)
            assert torch.equal(torch.autograd.grad(out[1], leaves[i], dh)[0], alone[i])


def test_gradients_against_differences():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w, b, dr, dh = make(4, 24, torch.float32, torch.float32, seed=8)
    for t in (x, r, w, b):
        t.requires_grad_()
    got = torch.autograd.grad(dgm.layer_norm_residual(x, r, w, b, residual_scale=0.7), (x, r, w, b), (dr, dh))
    leaves = [t.detach().double() for t in (x, r, w, b)]

    def loss(ls):
        f = Form(*ls, 0.7)
        return float((f.t * dr.double()).sum() + (f.h * dh.double()).sum())
    for k, g in enumerate(got):
        flat = g.flatten()
        for i in range(0, flat.numel(), max(1, flat.numel() // 7)):
            step = 1e-5
            ls = [t.clone() for t in leaves]
            ls[k].view(-1)[i] += step
            up = loss(ls)
            ls[k].view(-1)[i] -= 2 * step
            # (the formula's third derivative times step^2, and 64-bit rounding over step, are below 1e-6)
            assert abs((up - loss(ls)) / (2 * step) - float(flat[i])) < 1e-4 * (1 + abs(float(flat[i])))


def test_large_means_and_constant_rows():
    """The variance is that of the differences from the mean: a mean 1000 times the spread keeps it, and constant rows
    give the bias."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    g = torch.Generator(device="cuda").manual_seed(2)
    x = 1000 + torch.randn((6, 3000), generator=g, device="cuda")
    f = Form(x, None, None, None, 1.0)
    close(dgm.layer_norm_residual(x)[1], f.h, f.h_mag, 128)
    b = torch.randn(3000, generator=g, device="cuda")
    x = torch.full((3, 3000), 2.0, device="cuda")
    assert torch.equal(dgm.layer_norm_residual(x, bias=b)[1], b.expand(3, 3000))
    x = torch.zeros((2, 40), device="cuda", dtype=torch.bfloat16)
    r, h = dgm.layer_norm_residual(x, eps=0.0)
    assert bool(torch.isnan(h).all())                      # (0 / 0, as the formula has it)
    for bad in (float("nan"), float("inf")):
        x = torch.randn((3, 300), generator=g, device="cuda")
        clean = dgm.layer_norm_residual(x)[1]
        x[1, 7] = bad
        h = dgm.layer_norm_residual(x)[1]
        assert bool(torch.isnan(h[1]).any()) and torch.equal(h[[0, 2]], clean[[0, 2]])


@pytest.mark.parametrize("T,H", [(1, 1), (3, 33), (5, 40), (64, 7168), (70, 96), (2, 8200), (300, 2880), (258, 7168), (4, 5001), (1, 16384)])
def test_mxfp4_rows(T, H):
    """Bit for bit mxfp4_quantize of the rounded h, in one launch or two."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for wdt in (torch.bfloat16, torch.float32):
        x, r, w, b, *_ = make(T, H, torch.bfloat16, wdt, seed=H)
        want_r, want_h = dgm.layer_norm_residual(x, r, w, b)
        got_r, got_h, rows = dgm.layer_norm_residual(x, r, w, b, quant="mxfp4")
        assert torch.equal(got_r, want_r) and torch.equal(got_h, want_h)
        want = dgm.mxfp4_quantize(want_h)
        assert torch.equal(rows[0], want[0]) and torch.equal(rows[1], want[1])
    x[T // 2, H // 2] = float("nan")
    _, h, rows = dgm.layer_norm_residual(x, quant="mxfp4")
    want = dgm.mxfp4_quantize(h)
    assert torch.equal(rows[0], want[0]) and torch.equal(rows[1], want[1]) and bool((rows[1][T // 2] == 255).any())


@pytest.mark.parametrize("dtype", DT)
def test_strides_and_outputs(dtype):
    """Padded, unaligned and transposed rows, outputs over inputs' own rows and in padded memory."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w, b, dr, dh = make(40, 200, dtype, dtype, seed=1)
    want = dgm.layer_norm_residual(x, r, w, b, 0.5)
    grads = dgm.layer_norm_residual_backward(dr, dh, x, r, *dgm.layer_norm_residual_forward(x, r, w, b, 0.5)[2:], w, b, 0.5)

    def padded(t, left):
        big = torch.full((t.size(0), t.size(1) + 24), 9.0, dtype=dtype, device="cuda")
        big[:, left:left + t.size(1)] = t
        return big[:, left:left + t.size(1)]
    for lay in (lambda t: padded(t, 8), lambda t: padded(t, 3), lambda t: t.t().contiguous().t()):
        xs, rs = lay(x), lay(r)
        got = dgm.layer_norm_residual(xs, rs, w, b, 0.5)
        f = Form(x, r, w, b, 0.5)
        close(got[0], f.t, f.t_mag, 128)
        close(got[1], f.h, f.h_mag, 128)
        back = dgm.layer_norm_residual_backward(lay(dr), lay(dh), xs, rs, *dgm.layer_norm_residual_forward(xs, rs, w, b, 0.5)[2:], w, b, 0.5)
        for a, (name, (value, mag)) in zip(back, [(n, f.grads(dr, dh)[n]) for n in ("x", "residual", "weight", "bias")]):
            close(a, value, mag, 384 + (40 if name in ("weight", "bias") else 0))
    xs, rs = x.clone(), r.clone()
    got = dgm.layer_norm_residual(xs, rs, w, b, 0.5, residual_out=rs, out=xs)
    assert got[0] is rs and got[1] is xs and torch.equal(rs, want[0]) and torch.equal(xs, want[1])
    o1, o2 = torch.full((41, 216), 5.0, dtype=dtype, device="cuda"), torch.full((41, 216), 5.0, dtype=dtype, device="cuda")
    dgm.layer_norm_residual(x, r, w, b, 0.5, residual_out=o1[:40, :200], out=o2[:40, :200])
    assert torch.equal(o1[:40, :200], want[0]) and torch.equal(o2[:40, :200], want[1])
    assert bool((o1[40:] == 5).all()) and bool((o1[:, 200:] == 5).all()) and bool((o2[40:] == 5).all()) and bool((o2[:, 200:] == 5).all())
    assert all(torch.equal(p, q) for p, q in zip(grads, dgm.layer_norm_residual_backward(
        dr, dh, x, r, *dgm.layer_norm_residual_forward(x, r, w, b, 0.5)[2:], w, b, 0.5)))        # (the same bits again)
    wide = torch.stack([w, w], 1)[:, 0]                                                           # (a strided weight)
    assert torch.equal(dgm.layer_norm_residual(x, r, wide, b, 0.5)[1], want[1])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("left", [1, 2, 8])
def test_rows_of_any_length_between_others(dtype, left):
    """Rows that start and end anywhere, beside NaN that no row may read and values that none may write over."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for H in (1, 2, 5, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 31, 511, 513, 1027, 8193, 9001):
        x, r, w, b, dr, dh = make(3, H, dtype, dtype, seed=H)
        f = Form(x, r, w, b, 0.5)

        def within(t, fill):
            big = torch.full((5, H + left + 9), fill, dtype=dtype, device="cuda")
            view = big[1:4, left:left + H]
            view.copy_(t)
            return view, big
        xs, rs, drs, dhs = (within(t, float("nan"))[0] for t in (x, r, dr, dh))
        ws, bs = (torch.full((H + left + 9,), float("nan"), dtype=dtype, device="cuda")[left:left + H].copy_(t) for t in (w, b))
        (o1, all1), (o2, all2) = within(torch.zeros_like(x), 5.0), within(torch.zeros_like(x), 5.0)
        dgm.layer_norm_residual(xs, rs, ws, bs, 0.5, residual_out=o1, out=o2)
        close(o1, f.t, f.t_mag, 128)
        close(o2, f.h, f.h_mag, 128)
        for o, big in ((o1, all1), (o2, all2)):
            o.fill_(5.0)
            assert bool((big == 5.0).all()), H
        back = dgm.layer_norm_residual_backward(drs, dhs, xs, rs, *dgm.layer_norm_residual_forward(xs, rs, ws, bs, 0.5)[2:], ws, bs, 0.5)
        want = f.grads(dr, dh)
        for t, name in zip(back, ("x", "residual", "weight", "bias")):
            close(t, *want[name], 384 + (3 if name in ("weight", "bias") else 0))


def test_shared_leaves_no_rows_and_offsets():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, _, w, b, dr, dh = make(30, 64, torch.float32, torch.float32, seed=6)
    x.requires_grad_()
    r, h = dgm.layer_norm_residual(x, x, w, b, residual_scale=0.5)            # x is its own residual
    got = torch.autograd.grad((r, h), x, (dr, dh))[0]
    d = x.detach()
    parts = dgm.layer_norm_residual_backward(dr, dh, d, d, *dgm.layer_norm_residual_forward(d, d, w, b, 0.5)[2:], w, b, 0.5)
    assert torch.equal(got, parts[0] + parts[1])
    row = torch.randn((1, 64), device="cuda", requires_grad=True)             # one residual row for all tokens
    r, h = dgm.layer_norm_residual(d, row.expand(30, 64), w, b)
    got = torch.autograd.grad(h, row, dh)[0]
    one = dgm.layer_norm_residual_backward(None, dh, d, row.detach().expand(30, 64),
                                           *dgm.layer_norm_residual_forward(d, row.detach().expand(30, 64), w, b)[2:], w, b)[1]
    assert torch.allclose(got, one.sum(0, keepdim=True), rtol=0, atol=float(one.abs().sum(0).max()) * 30 * U)
    e = torch.zeros((0, 64), device="cuda", requires_grad=True)
    wl = torch.ones(64, device="cuda", requires_grad=True)
    r, h = dgm.layer_norm_residual(e, None, wl, residual_scale=2.0)
    gx, gw = torch.autograd.grad((r, h), (e, wl), (torch.zeros_like(r), torch.zeros_like(h)))
    assert gx.shape == (0, 64) and not bool(gw.any())
    big = torch.zeros((20, 1 << 27), dtype=torch.bfloat16, device="cuda")[:, :512]          # rows 2^28 bytes apart
    src = torch.randn((20, 512), device="cuda").to(torch.bfloat16)
    big.copy_(src)
    assert torch.equal(dgm.layer_norm_residual(big)[1], dgm.layer_norm_residual(src)[1])


def test_streams_and_graphs():
    """Forward and backward replayed from a graph against eager calls, on another stream at the same time."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w, b, dr, dh = make(100, 1024, torch.bfloat16, torch.float32, seed=12)

    def run():
        ro, h, mean, rstd = dgm.layer_norm_residual_forward(x, r, w, b, 0.5)
        return (ro, h) + dgm.layer_norm_residual_backward(dr, dh, x, r, mean, rstd, w, b, 0.5)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        x.normal_()
        dh.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = run()
        eager = run()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) and torch.equal(p, o) for p, q, o in zip(got, eager, other)), i
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="under graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            dgm.layer_norm_residual(x, r, w, b)
    out = dgm.layer_norm_residual(x, r, w, b)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out[1].sum(), x, create_graph=True)


def test_saved_tensors_that_hooks_bring_back():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w, b, dr, dh = make(20, 128, torch.bfloat16, torch.bfloat16, seed=15)
    for t in (x, r, w, b):
        t.requires_grad_()
    want = torch.autograd.grad(dgm.layer_norm_residual(x, r, w, b, 0.5), (x, r, w, b), (dr, dh))
    with torch.autograd.graph.save_on_cpu():
        out = dgm.layer_norm_residual(x, r, w, b, 0.5)
    got = torch.autograd.grad(out, (x, r, w, b), (dr, dh))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    out = dgm.layer_norm_residual(x, r, w, b, 0.5)
    with torch.no_grad():
        dgm.layer_norm_residual(r, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out, x, (dr, dh))
