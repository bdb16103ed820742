"""mega_moe_block with an MXFP4 dense expert and with layer norms: its parts, one by one, and the same from a graph."""
import pytest
import torch

from tests.gpu_common import need_gpu
from tests.test_gpu_block import E, H, TOPK, setup

pytestmark = pytest.mark.gpu
INNER = 352


def dense(dgm, rnd):
    return dgm.mxfp4_quantize(rnd(2 * INNER, H, scale=0.05)), dgm.mxfp4_quantize(rnd(H, INNER, scale=0.05))


@pytest.mark.parametrize("tokens", [0, 1, 7, 64])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_block_is_its_parts(tokens, norm):
    need_gpu()
    dgm, l1, l2, int8, b, w, rnd = setup("mxfp4")
    x, res = rnd(tokens, H), rnd(tokens, H)
    biases = dict(norm_bias=rnd(H, scale=0.1), next_bias=rnd(H, scale=0.1)) if norm == "layer" else {}
    for shared in (dense(dgm, rnd), int8, None):
        stats = torch.zeros(E, dtype=torch.int32, device="cuda")
        r, h = dgm.mega_moe_block(x, w["norm"], w["router"], l1, l2, b, residual=res, shared_expert=shared, residual_scale=0.5,
                                  next_weight=w["next"], norm=norm, cumulative_local_expert_recv_stats=stats, **biases)
        assert r.shape == h.shape == (tokens, H) and int(stats.sum()) == tokens * TOPK
        if tokens == 0:
            continue
        if norm == "layer":
            s, h1 = dgm.layer_norm_residual(x, res, w["norm"], biases["norm_bias"], eps=1e-6)
        else:
            s, h1 = dgm.rms_norm_residual(x, res, pre_weight=w["norm"])
        y = torch.empty_like(h1)
        dgm.mxfp4_mega_moe_from_bf16(y, h1, w["router"], l1, l2, b)
        if shared is not None:
            mx = shared[0][0].dtype == torch.uint8
            act = torch.empty((tokens, INNER if mx else shared[1][0].size(1)), dtype=torch.bfloat16, device="cuda")
            cast, product = (dgm.mxfp4_quantize, dgm.mxfp4_gemm_nt) if mx else (dgm.quantization_qoq_fused.per_token_cast_to_int8, dgm.int8_gemm_nt)
            product(cast(h1), shared[0], act, activation="swiglu")
            product(cast(act), shared[1], y, c=y)
        if norm == "layer":
            want = dgm.layer_norm_residual(y, s, w["next"], biases["next_bias"], residual_scale=0.5, eps=1e-6)
        else:
            want = dgm.rms_norm_residual(y, s, pre_weight=w["next"], residual_scale=0.5)
        assert torch.equal(r, want[0]) and torch.equal(h, want[1])
        alone = dgm.mega_moe_block(x, w["norm"], w["router"], l1, l2, b, residual=res, shared_expert=shared, residual_scale=0.5, norm=norm,
                                   **{k: v for k, v in biases.items() if k == "norm_bias"})
        assert torch.equal(alone[0], r) and alone[1] is None


def test_in_a_graph():
    need_gpu()
    dgm, l1, l2, _, b, w, rnd = setup("mxfp4")
    shared, x, bias = dense(dgm, rnd), rnd(20, H), rnd(H, scale=0.1)
    run = lambda: dgm.mega_moe_block(x, w["norm"], w["router"], l1, l2, b, residual=x, shared_expert=shared, next_weight=w["next"],
                                     norm="layer", norm_bias=bias)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(3):
        x.copy_(rnd(20, H))
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager)), i


def test_a_training_step():
    """Layer norm, two linear layers on MXFP4 products and the residual add back: the gradients are those of the parts
    called one by one, and a second step of the same gives the same bits."""
    need_gpu()
    import hopper_megamoe_basedondeepgemm_amd as dgm
    torch.manual_seed(0)
    x = torch.randn((96, 128), device="cuda").to(torch.bfloat16).requires_grad_()
    g, b = torch.ones(128, device="cuda", requires_grad=True), torch.zeros(128, device="cuda", requires_grad=True)
    w1 = (torch.randn((256, 128), device="cuda") * 0.1).requires_grad_()
    w2 = (torch.randn((128, 256), device="cuda") * 0.1).requires_grad_()
    leaves = (x, g, b, w1, w2)

    def step():
        s, h = dgm.layer_norm_residual(x, weight=g, bias=b)
        y = dgm.mxfp4_linear(dgm.mxfp4_linear(h, w1), w2)
        return dgm.layer_norm_residual(y, s, g, b, residual_scale=0.5)
    dr, dh = torch.randn_like(x), torch.randn_like(x)
    out = step()
    got = torch.autograd.grad(out, leaves, (dr, dh))
    assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad(step(), leaves, (dr, dh))))
    X, G, B, W1, W2 = (t.detach() for t in leaves)
    s, h, m1, r1 = dgm.layer_norm_residual_forward(X, None, G, B)
    u, ht, w1t = dgm.mxfp4_linear_forward(h, W1)
    y, ut, w2t = dgm.mxfp4_linear_forward(u, W2)
    r, h2, m2, r2 = dgm.layer_norm_residual_forward(y, s, G, B, 0.5)
    assert torch.equal(out[0], r) and torch.equal(out[1], h2)
    dy, ds, dg2, db2 = dgm.layer_norm_residual_backward(dr, dh, y, s, m2, r2, G, B, 0.5)
    du, dw2 = dgm.mxfp4_linear_backward(dy, ut, w2t, u.shape, W2.shape, W2.dtype)
    dhh, dw1 = dgm.mxfp4_linear_backward(du, ht, w1t, h.shape, W1.shape, W1.dtype)
    dx, _, dg1, db1 = dgm.layer_norm_residual_backward(ds, dhh, X, None, m1, r1, G, B)
    for a, e in zip(got, (dx, dg1 + dg2, db1 + db2, dw1, dw2)):
        assert torch.equal(a, e)
