"""rms_norm_residual and its gradients against the formulas in 64 bits.

Tolerances: every element may be off by half a step of its type (finfo.eps / 2 of the value) for the last
rounding, and by C 2^-24 of the same formula over absolute values for the fp32 arithmetic. C counts
roundings: a mean over H squares adds at most 16 terms per thread, 4 by lane exchange, 3 wave parts and 15
wave sums (< 40), halved by the root; with the products around it every value is within 64. A gradient
holds two such means and the recomputed row: 256. A sum over T rows adds at most T more."""
import numpy as np
import pytest
import torch

from tests.gpu_common import need_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6


def close(got, ref, mag, c):
    """|got - ref| <= half a step of got's type + c 2^-24 mag (and the least normal number)"""
    fi = torch.finfo(got.dtype)
    tol = ref.abs() * (fi.eps / 2) + c * U * mag * (1 + fi.eps) + fi.tiny
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((off / tol).max()), got.dtype)


class Form:
    """The formulas in 64 bits, and the same over absolute values (for the error of fp32 sums)."""

    def __init__(self, x, r, w1, w2, g, sigmoid, s, eps=EPS):
        d = lambda t: None if t is None else t.detach().double()
        x, r, w1, w2, g = d(x), d(r), d(w1), d(w2), d(g)
        self.w1, self.w2, self.s, self.sigmoid = w1, w2, s, sigmoid
        self.rstd1 = torch.rsqrt(x.square().mean(1, keepdim=True) + eps) if w1 is not None else torch.ones_like(x[:, :1])
        self.z = x * self.rstd1
        self.n = self.z * w1 if w1 is not None else self.z
        self.a = torch.ones_like(x) if g is None else (torch.sigmoid(g) if sigmoid else g).expand_as(x)
        self.gshape = None if g is None else g.shape
        res = 0 if r is None else r
        self.t = res + s * self.a * self.n
        self.t_mag = (0 if r is None else r.abs()) + abs(s) * self.a.abs() * self.n.abs()
        self.rstd2 = torch.rsqrt(self.t.square().mean(1, keepdim=True) + eps)
        self.u = self.t * self.rstd2
        # (the mean of t^2 takes t's absolute error, 2 t dt, twice over the root)
        self.u_mag = self.t_mag * self.rstd2 + self.u.abs() * (self.t.abs() * self.t_mag).mean(1, keepdim=True) * self.rstd2 ** 2
        self.h = self.u * w2 if w2 is not None else None
        self.h_mag = self.u_mag * w2.abs() if w2 is not None else None

    def over(self, v):
        """v reduced to the gate's shape"""
        if len(self.gshape) == 1:
            return v.sum(0)
        return v.sum(1, keepdim=True) if self.gshape[1] == 1 and v.size(1) != 1 else v

    def grads(self, dr, dh):
        """{name: (value, magnitude)}"""
        out = {}
        R = torch.zeros_like(self.t) if dr is None else dr.double()
        Rm = R.abs()
        if dh is not None:
            D = dh.double()
            du = D * self.w2
            m = (du * self.u).mean(1, keepdim=True)
            mm = (du.abs() * self.u_mag).mean(1, keepdim=True)
            out["pre"] = ((D * self.u).sum(0), (D.abs() * self.u_mag).sum(0))
            spread = (self.u.abs() * self.u_mag).mean(1, keepdim=True) + 1     # rstd2's own error
            Rm = Rm + self.rstd2 * (du.abs() + self.u_mag * m.abs() + self.u_mag * mm) * spread
            R = R + self.rstd2 * (du - self.u * m)
        out["residual"] = (R, Rm)
        dn, dnm = self.s * R * self.a, abs(self.s) * Rm * self.a.abs()
        if self.gshape is not None:
            k = self.a * (1 - self.a) if self.sigmoid else 1.0
            # 1 - sigmoid is off by 2^-24 of 1, not of itself
            km = self.a.abs() if self.sigmoid else 1.0
            out["gate"] = (self.over(self.s * R * self.n * k), self.over(abs(self.s) * Rm * self.n.abs() * km))
        if self.w1 is not None:
            out["post"] = ((dn * self.z).sum(0), (dnm * self.z.abs()).sum(0))
            dz, dzm = dn * self.w1, dnm * self.w1.abs()
            m = (dz * self.z).mean(1, keepdim=True)
            mm = (dzm * self.z.abs()).mean(1, keepdim=True)
            dn, dnm = self.rstd1 * (dz - self.z * m), self.rstd1 * (dzm + self.z.abs() * mm)
        out["x"] = (dn, dnm)
        return out


def make(T, H, dtype, wdtype, post, pre, gate, residual, seed=0, spread=1.0):
    torch.manual_seed(seed)                 # (for what a test draws after this)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    x = (rnd(T, H) * spread).to(dtype)
    r = rnd(T, H).to(dtype) if residual else None
    w1 = (1 + 0.2 * rnd(H)).to(wdtype) if post else None
    w2 = (1 + 0.2 * rnd(H)).to(wdtype) if pre else None
    shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[gate]
    gt = rnd(*shape).to(dtype) if shape else None
    return x, r, w1, w2, gt


def check_forward(x, r, w1, w2, gt, sigmoid, s, got_r, got_h):
    f = Form(x, r, w1, w2, gt, sigmoid, s)
    if got_r is not x:
        close(got_r, f.t, f.t_mag, 64)
    if w2 is not None:
        close(got_h, f.h, f.h_mag, 64)
    else:
        assert got_h is None
    return f


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 100), (4, 512), (3, 513), (9, 1024), (2, 1032), (7, 2880), (2, 4096), (1, 4104),
          (3, 8192), (2, 8200), (2, 12345), (1, 16384),
          (300, 512), (257, 1000), (300, 2048), (258, 2880), (260, 7168), (257, 9000), (300, 33)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_forward_shapes(T, H, dtype):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for post, pre, gate, residual, sigmoid, s, wdt in ((0, 1, "none", 0, False, 1.0, dtype), (0, 1, "none", 1, False, 1.0, dtype),
                                                       (1, 1, "channel", 1, False, 0.22, dtype),
                                                       (1, 1, "token", 1, True, 1.0, torch.float32),
                                                       (1, 0, "full", 1, True, -0.5, dtype), (0, 0, "none", 1, False, 2.0, dtype),
                                                       (1, 1, "full", 0, False, 0.5, torch.float32)):
        x, r, w1, w2, gt = make(T, H, dtype, wdt, post, pre, gate, residual, seed=T * H)
        got_r, got_h = dgm.rms_norm_residual(x, r, w1, w2, gt, sigmoid, s)
        check_forward(x, r, w1, w2, gt, sigmoid, s, got_r, got_h)


def test_plain_pre_norm_returns_its_input():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, _, _, w2, _ = make(4, 256, torch.bfloat16, torch.bfloat16, 0, 1, "none", 0)
    r, h = dgm.rms_norm_residual(x, pre_weight=w2)
    assert r is x
    r, h = dgm.rms_norm_residual(x)
    assert r is x and h is None
    xg = x.clone().requires_grad_()
    r, h = dgm.rms_norm_residual(xg, pre_weight=w2)
    assert r is xg
    (g,) = torch.autograd.grad(h.float().sum() + 2 * r.float().sum(), xg)
    f = Form(x, None, None, w2, None, False, 1.0)
    v, m = f.grads(2 * torch.ones_like(x), torch.ones_like(x))["residual"]
    # (autograd adds the two parts in bf16: one more rounding of the part and of the sum)
    assert bool(((g.double() - v).abs() <= 2.0 ** -8 * (v.abs() + (v - 2).abs()) * 1.01 + 256 * U * m).all())


def test_no_rows():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w1, w2, gt = make(0, 256, torch.bfloat16, torch.float32, 1, 1, "channel", 1)
    leaves = [t.requires_grad_() for t in (x, r, w1, w2, gt)]
    got_r, got_h = dgm.rms_norm_residual(*leaves)
    assert got_r.shape == got_h.shape == (0, 256)
    grads = torch.autograd.grad((got_r, got_h), leaves, (torch.ones_like(got_r), torch.ones_like(got_h)))
    for t, g in zip(leaves, grads):
        assert g.shape == t.shape and g.dtype == t.dtype and not bool(g.float().any())


@pytest.mark.parametrize("T,H", [(1, 8), (1, 4096), (5, 1), (6, 100), (3, 513), (700, 64), (37, 1024), (1300, 320), (17, 2880),
                                 (12, 5000), (9, 8192), (5, 10001), (4, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gradients(T, H, dtype):
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    for post, pre, gate, residual, sigmoid, s, wdt in ((0, 1, "none", 1, False, 1.0, dtype), (1, 1, "channel", 1, False, 0.22, dtype),
                                                       (1, 1, "channel", 1, True, 1.0, torch.float32),
                                                       (1, 1, "token", 1, True, 1.0, torch.float32),
                                                       (0, 1, "token", 1, False, 0.7, dtype),
                                                       (1, 1, "full", 0, True, -0.5, dtype), (1, 0, "none", 1, False, 2.0, dtype)):
        x, r, w1, w2, gt = make(T, H, dtype, wdt, post, pre, gate, residual, seed=T + H)
        ins = dict(x=x, residual=r, post=w1, pre=w2, gate=gt)
        leaves = {k: v.requires_grad_() for k, v in ins.items() if v is not None}
        got_r, got_h = dgm.rms_norm_residual(x, r, w1, w2, gt, sigmoid, s)
        f = check_forward(x, r, w1, w2, gt, sigmoid, s, got_r, got_h)
        dr = torch.randn_like(got_r)
        dh = None if got_h is None else torch.randn_like(got_h)
        outs, douts = ([got_r, got_h], [dr, dh]) if got_h is not None else ([got_r], [dr])
        grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), douts)))
        want = f.grads(dr, dh)
        if r is None:
            del want["residual"]
        assert set(want) == set(grads)
        for k, (v, m) in want.items():
            assert grads[k].shape == ins[k].shape and grads[k].dtype == ins[k].dtype
            over = T if v.dim() == 1 else H if v.shape != f.t.shape else 0
            close(grads[k], v, m, 256 + over)


def test_gradients_against_differences():
    """dL along a direction against central differences of the formula in 64 bits."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w1, w2, gt = make(6, 96, torch.float32, torch.float32, 1, 1, "channel", 1, seed=5)
    leaves = [t.requires_grad_() for t in (x, r, w1, w2, gt)]
    got_r, got_h = dgm.rms_norm_residual(*leaves, True, 0.3)
    dr, dh = torch.randn_like(got_r), torch.randn_like(got_h)
    grads = torch.autograd.grad((got_r, got_h), leaves, (dr, dh))

    def loss(v):
        f = Form(*v, True, 0.3)
        return float((f.t * dr.double()).sum() + (f.h * dh.double()).sum())
    base = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        way = torch.randn_like(base[i])
        e = 1e-5
        up = [b + e * way if j == i else b for j, b in enumerate(base)]
        dn = [b - e * way if j == i else b for j, b in enumerate(base)]
        diff = (loss(up) - loss(dn)) / (2 * e)
        got = float((g.double() * way).sum())
        # central difference: e^2 of the third derivative (values of order 10 here) and 64-bit cancellation,
        # both below 1e-7 of the sum of magnitudes; the gradient's own 2^-24 errors: 512 of them at most
        assert abs(diff - got) <= 512 * U * float((g.double().abs() * way.abs()).sum() + 10), (i, diff, got)


def test_one_sided_gradients():
    """Only r, or only h, reaches the loss; inputs that need no gradient."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w1, w2, gt = make(33, 256, torch.float32, torch.float32, 1, 1, "token", 1, seed=3)
    for use_r, use_h in ((True, False), (False, True)):
        x_ = x.detach().requires_grad_()
        g_ = gt.detach().requires_grad_()
        got_r, got_h = dgm.rms_norm_residual(x_, r, w1, w2, g_, False, 0.5)
        d = torch.randn_like(x)
        out = got_r if use_r else got_h
        gx, gg = torch.autograd.grad(out, (x_, g_), d)
        want = Form(x, r, w1, w2, gt, False, 0.5).grads(d if use_r else None, d if use_h else None)
        close(gx, *want["x"], 256)
        close(gg, *want["gate"], 512)


@pytest.mark.parametrize("H", [100, 512, 2880, 7168, 8200])
def test_int8_rows(H):
    """q, sf are per_token_cast_to_int8 of the returned h bit for bit; a zero row has zero codes."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, _, w2, _ = make(9, H, torch.bfloat16, torch.bfloat16, 0, 1, "none", 1, seed=H)
    x[4], r[4] = 0, 0
    got_r, h, (q, sf) = dgm.rms_norm_residual(x, r, pre_weight=w2, quant="int8")
    check_forward(x, r, None, w2, None, False, 1.0, got_r, h)
    K = H // 128 * 128
    if K == H:
        q2, sf2 = dgm.quantization_qoq_fused.per_token_cast_to_int8(h)
        assert torch.equal(q, q2) and torch.equal(sf, sf2[:, 0])
    else:
        # (on the CPU: torch's division by a scalar on the GPU is a product with its rounded reciprocal)
        v = h.float().cpu().numpy()
        s = np.maximum(np.abs(v).max(1), np.float32(1e-30)) / np.float32(127)
        assert (sf.cpu().numpy() == s).all()
        assert (q.cpu().numpy() == np.clip(np.rint(v / s[:, None]), -127, 127)).all()
    assert not bool(q[4].any()) and q.dtype == torch.int8 and sf.shape == (9,)


def test_int8_rows_of_any_value():
    """Rows over all of bf16: each magnitude as a row's largest with all kinds of values below it, denormal, infinite and
    NaN ones included, cast as per_token_cast_to_int8 casts them."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    cast = dgm.quantization_qoq_fused.per_token_cast_to_int8
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.ones((1, 1024), device="cuda").bfloat16()
    x[0, 1::2] = -1                                       # (mean square 1, eps 0: h is the weight)
    for top in [0.0] + [2.0 ** e * (1 + f / 128) for e in range(-133, 128, 3) for f in (0, 37, 126, 127)] + [float("inf"), float("nan")]:
        scale = top if 0 < top < float("inf") else 3.0
        w = scale * torch.rand(1024, generator=g, device="cuda", dtype=torch.float64)
        w[:512] *= torch.linspace(0, 1, 512, device="cuda", dtype=torch.float64)
        w[512:640] = (torch.arange(128, device="cuda") - 0.5) / 127 * scale          # (halves of a step)
        w[5] = top
        w = w.float().bfloat16()
        _, h, (q, sf) = dgm.rms_norm_residual(x, pre_weight=w, eps=0.0, quant="int8")
        assert torch.equal(h.abs().nan_to_num(7.0), w[None].abs().nan_to_num(7.0)), top
        want, want_sf = cast(h)
        assert torch.equal(sf, want_sf[:, 0]) and torch.equal(q, want), top


def test_strides_alignment_and_places():
    """Row strides, misaligned rows, transposed and expanded inputs, outputs over the inputs' rows: the
    same values as from plain inputs, and nothing beside the rows written."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    T, H = 5, 640
    x, r, w1, w2, gt = make(T, H, torch.bfloat16, torch.bfloat16, 1, 1, "full", 1, seed=1)
    want = dgm.rms_norm_residual(x, r, w1, w2, gt, True, 0.5)

    def same(got):
        check_forward(x, r, w1, w2, gt, True, 0.5, *got)

    for shift in (0, 1, 8):
        wide = lambda t: torch.full((T, H + 24), 7.0, dtype=t.dtype, device="cuda")[:, shift:shift + H].copy_(t)
        same(dgm.rms_norm_residual(wide(x), wide(r), w1, w2, wide(gt), True, 0.5))
    turned = lambda t: t.t().contiguous().t()
    same(dgm.rms_norm_residual(turned(x), turned(r), w1, w2, turned(gt), True, 0.5))
    one = torch.randn(H, device="cuda").bfloat16()
    a = dgm.rms_norm_residual(x, one.expand(T, H), w1, w2, gt, True, 0.5)
    b = dgm.rms_norm_residual(x, one.repeat(T, 1), w1, w2, gt, True, 0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    every = torch.stack([w1, w2], 1)                      # strided weights
    same(dgm.rms_norm_residual(x, r, every[:, 0], every[:, 1], gt, True, 0.5))
    # in place: r over residual, h over x
    big_x, big_r = (torch.full((T + 2, H + 8), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    xi, ri = big_x[1:-1, :H].copy_(x), big_r[1:-1, :H].copy_(r)
    got = dgm.rms_norm_residual(xi, ri, w1, w2, gt, True, 0.5, residual_out=ri, out=xi)
    assert got[0] is ri and got[1] is xi and torch.equal(ri, want[0]) and torch.equal(xi, want[1])
    for big in (big_x, big_r):
        assert bool((big[0] == 3).all() and (big[-1] == 3).all() and (big[:, H:] == 3).all())
    with pytest.raises(ValueError, match="overlaps an input"):
        dgm.rms_norm_residual(big_x[:T, :H], r, w1, w2, gt, residual_out=big_x[1:T + 1, :H])
    with pytest.raises(ValueError, match="outputs overlap"):
        dgm.rms_norm_residual(x, r, w1, w2, gt, residual_out=xi, out=xi)
    with pytest.raises(ValueError, match="no gradient"):
        dgm.rms_norm_residual(x.clone().requires_grad_(), r, w1, w2, gt, residual_out=ri)


def test_shared_and_broadcast_leaves():
    """One leaf in several places, expanded residual and gate: their gradients are the sums over the places."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    T, H = 12, 96
    x, _, w1, _, _ = make(T, H, torch.float32, torch.float32, 1, 0, "none", 0, seed=4)
    row, g = torch.randn(H, device="cuda"), torch.randn(1, 1, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, row, w1, g)]
    lx, lr, lw, lg = leaves
    got = dgm.rms_norm_residual(lx, lr.expand(T, H), lw, lw, lg.expand(T, 1), True, 0.5)
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    gx, gr, gw, gg = torch.autograd.grad(got, leaves, (dr, dh))
    want = Form(x, row.expand(T, H), w1, w1, g.expand(T, 1), True, 0.5).grads(dr, dh)
    close(gx, *want["x"], 256)
    close(gr, *(v.sum(0) for v in want["residual"]), 256 + T)
    close(gw, want["post"][0] + want["pre"][0], want["post"][1] + want["pre"][1], 256 + 2 * T)
    close(gg, *(v.sum(0, keepdim=True) for v in want["gate"]), 256 + H + T)
    both = x.clone().requires_grad_()
    r, h = dgm.rms_norm_residual(both, both, pre_weight=w1)
    (gb,) = torch.autograd.grad((r, h), both, (dr, dh))
    want = Form(x, x, None, w1, None, False, 1.0).grads(dr, dh)
    close(gb, want["x"][0] + want["residual"][0], want["x"][1] + want["residual"][1], 257)


def test_memory_that_moves_between_the_passes():
    """Parameters and activations whose storage is replaced between forward and backward (as sharded training
    does), and inputs that are read as copies."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w1, w2, gt = make(9, 160, torch.bfloat16, torch.float32, 1, 1, "channel", 1, seed=8)
    dr, dh = torch.randn_like(x), torch.randn_like(x)

    def grads(move, turn):
        t = lambda v: v.t().contiguous().t() if turn and v.dim() == 2 else v.clone()
        leaves = [t(v).requires_grad_() for v in (x, r, w1, w2, gt)]
        got = dgm.rms_norm_residual(*leaves, True, 0.5)
        if move:
            for v in leaves:
                v.data = v.data.clone(memory_format=torch.preserve_format)
            torch.cuda.synchronize()
        return torch.autograd.grad(got, leaves, (dr, dh), retain_graph=True), torch.autograd.grad(got, leaves, (dr, dh))
    want, again = grads(False, False)
    for case in ((False, True), (True, False), (True, True)):
        for got in grads(*case):
            assert all(torch.equal(a, b) for a, b in zip(want, got)), case
    assert all(torch.equal(a, b) for a, b in zip(want, again))


@pytest.mark.parametrize("way", ["offload", "recompute", "moved"])
@pytest.mark.parametrize("post,pre", [(1, 1), (0, 1), (1, 0), (0, 0)])
def test_saved_tensors_that_hooks_bring_back(way, post, pre):
    """Tensors saved for the backward pass that come back in other memory and other strides, the rstd rows among them:
    the gradients are those of the plain call, bit for bit."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    from torch.utils.checkpoint import checkpoint
    x, r, w1, w2, gt = make(37, 200, torch.bfloat16, torch.float32, post, pre, "full", 1, seed=9)
    wide = torch.randn((37, 320), device="cuda").to(torch.bfloat16)
    wide[:, 40:240] = x
    dr, dh = torch.randn_like(x), torch.randn_like(x)

    def grads(how):
        base, leaves = wide.clone().requires_grad_(), [v if v is None else v.clone().requires_grad_() for v in (r, w1, w2, gt)]

        def run(base, *rest):
            return dgm.rms_norm_residual(base[:, 40:240], *rest, True, 0.5)
        if how == "offload":
            with torch.autograd.graph.save_on_cpu():
                got = run(base, *leaves)
        elif how == "recompute":
            got = checkpoint(run, base, *leaves, use_reentrant=False)
        elif how == "moved":
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2
                                                          else t.clone()):
                got = run(base, *leaves)
        else:
            got = run(base, *leaves)
        keep = [torch.full((2, 37), 7.0, device="cuda") for _ in range(64)]     # (over rows that were given up)
        pairs = [(o, d) for o, d in zip(got, (dr, dh)) if o is not None]
        out = torch.autograd.grad([o for o, _ in pairs], [base] + [v for v in leaves if v is not None], [d for _, d in pairs])
        del keep
        return out
    for a, b in zip(grads("plain"), grads(way)):
        assert torch.equal(a, b)


def test_autograd_refusals():
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, _, _, w2, _ = make(4, 64, torch.float32, torch.float32, 0, 1, "none", 0)
    leaf = x.clone().requires_grad_()
    _, h = dgm.rms_norm_residual(leaf, pre_weight=w2)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(h.sum(), leaf, create_graph=True)
    _, h = dgm.rms_norm_residual(leaf * 1, pre_weight=w2)
    mid = leaf * 1
    _, h = dgm.rms_norm_residual(mid, pre_weight=w2)
    with torch.no_grad():
        mid.zero_()                                       # (an input changed behind the forward pass)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(h.sum(), leaf)
    with pytest.raises(RuntimeError, match="cpu"):
        dgm.rms_norm_residual(x, x.cpu())


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart, read and written."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    T, H, gap = 4, 512, (1 << 30) + 64
    big = torch.empty(gap * (T - 1) + H, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((T, H), (gap, 1))
    x, r, w1, w2, gt = make(T, H, torch.bfloat16, torch.float32, 1, 1, "token", 1, seed=6)
    far.copy_(x)
    want = dgm.rms_norm_residual_forward(x, r, w1, w2, gt, True, 0.5)
    got = dgm.rms_norm_residual_forward(far, r, w1, w2, gt, True, 0.5)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    a = dgm.rms_norm_residual_backward(dr, dh, x, r, *want[2:], w1, w2, gt, True, 0.5)
    b = dgm.rms_norm_residual_backward(dr, dh, far, r, *want[2:], w1, w2, gt, True, 0.5)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    dgm.rms_norm_residual(x, r, w1, w2, gt, True, 0.5, out=far)
    assert torch.equal(far, want[1])


def test_odd_values():
    """All-zero rows, rows of a large norm, infinities and NaN: as the formula has them, row by row."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w1, w2, _ = make(6, 256, torch.float32, torch.float32, 1, 1, "none", 1, seed=2)
    x[0], r[0] = 0, 0
    x[1] *= 1e15
    x[2, 3] = float("inf")
    x[3, 5] = float("nan")
    got_r, got_h = dgm.rms_norm_residual(x, r, w1, w2)
    f = Form(x, r, w1, w2, None, False, 1.0)
    assert not bool(got_r[0].any() or got_h[0].any())
    for k in (1, 4, 5):
        close(got_r[k], f.t[k], f.t_mag[k], 64)
        close(got_h[k], f.h[k], f.h_mag[k], 64)
    assert bool(torch.isnan(got_r[2, 3])) and bool(torch.isnan(got_r[3]).all()) and bool(torch.isnan(got_h[2:4]).all())
    keep = [c for c in range(256) if c != 3]
    assert torch.equal(got_r[2, keep], r[2, keep])        # rstd 0: the other elements add nothing


def test_repeats_streams_and_graph():
    """Same bits on every call, on another stream, and from a captured forward and backward replayed
    between eager calls."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    T, H = 700, 1024
    x, r, w1, w2, gt = make(T, H, torch.bfloat16, torch.float32, 1, 1, "channel", 1, seed=9)
    dr, dh = torch.randn_like(x), torch.randn_like(x)

    def both():
        got_r, got_h, a, b = dgm.rms_norm_residual_forward(x, r, w1, w2, gt, True, 0.5)
        return (got_r, got_h, *dgm.rms_norm_residual_backward(dr, dh, x, r, a, b, w1, w2, gt, True, 0.5))
    want = [t.clone() for t in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
        with pytest.raises(RuntimeError, match="no autograd under graph capture"):
            dgm.rms_norm_residual(x.detach().requires_grad_(), r, w1, w2)
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        now = both()
        assert all(torch.equal(a, b) for a, b in zip(held, now)), i


def test_saved_tensors_that_stay_on_the_cpu():
    """A hook that leaves a tensor on the CPU: refused before its address is read."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    x, r, w1, w2, gt = make(6, 96, torch.bfloat16, torch.float32, 1, 1, "token", 1, seed=4)
    for part in ((6, 96), (96,), (6, 1), (2, 6)):
        leaf = x.clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu() if t.shape == part else t):
            got = dgm.rms_norm_residual(leaf, r, w1, w2, gt)
        with pytest.raises(RuntimeError, match="cpu|GPU"):
            torch.autograd.grad(got, leaf, (torch.ones_like(x), torch.ones_like(x)))
