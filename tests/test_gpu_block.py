"""mega_moe_block: the operators around the layer run together as they are used."""
import numpy as np
import pytest
import torch

from tests.gpu_common import need_gpu

pytestmark = pytest.mark.gpu
E, H, I, TOPK, SHARED = 16, 512, 256, 4, 384
U = 2.0 ** -24


def setup(act_format="mxfp8", tokens=64):
    import hopper_megamoe_basedondeepgemm_amd as dgm
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s, scale=1.0: (torch.randn(s, generator=g, device="cuda") * scale).bfloat16()
    q = dgm.quantization_mxfp4_fused.quantize_to_mxfp4
    l1, l2 = dgm.transform_mxfp4_weights_for_mega_moe_fused(q(rnd(E, 2 * I, H, scale=0.05)), q(rnd(E, H, I, scale=0.05)))
    cast = dgm.quantization_qoq_fused.per_token_cast_to_int8
    shared = cast(rnd(2 * SHARED, H, scale=0.05)), cast(rnd(H, SHARED, scale=0.05))
    b = dgm.get_fused_symm_buffer_for_mega_moe(None, E, tokens, TOPK, H, I, act_format=act_format)
    w = dict(norm=1 + rnd(H, scale=0.1), post=1 + rnd(H, scale=0.1), next=1 + rnd(H, scale=0.1), router=rnd(E, H, scale=0.05))
    return dgm, l1, l2, shared, b, w, rnd


@pytest.mark.parametrize("tokens", [0, 1, 7, 64])
@pytest.mark.parametrize("act_format", ["mxfp8", "mxfp4"])
def test_block_is_its_parts(tokens, act_format):
    need_gpu()
    dgm, l1, l2, shared, b, w, rnd = setup(act_format)
    x, res, gate = rnd(tokens, H), rnd(tokens, H), rnd(tokens, 1)
    stats = torch.zeros(E, dtype=torch.int32, device="cuda")
    r, h = dgm.mega_moe_block(x, w["norm"], w["router"], l1, l2, b, residual=res, shared_expert=shared, post_weight=w["post"],
                              gate=gate, gate_sigmoid=True, residual_scale=0.5, next_weight=w["next"],
                              cumulative_local_expert_recv_stats=stats)
    assert r.shape == h.shape == (tokens, H) and int(stats.sum()) == tokens * TOPK
    if tokens == 0:
        return
    idx, logits = b.topk_idx[:tokens].clone(), b.logits[:tokens].clone()
    s, h1, rows = dgm.rms_norm_residual(x, res, pre_weight=w["norm"], quant="int8")
    y = torch.empty_like(h1)
    dgm.mxfp4_mega_moe_from_bf16(y, h1, w["router"], l1, l2, b)
    routed = y.clone()
    act = torch.empty((tokens, SHARED), dtype=torch.bfloat16, device="cuda")
    dgm.int8_gemm_nt(rows, shared[0], act, activation="swiglu")
    rows2 = dgm.quantization_qoq_fused.per_token_cast_to_int8(act)
    dgm.int8_gemm_nt(rows2, shared[1], y, c=y)
    want = dgm.rms_norm_residual(y, s, w["post"], w["next"], gate, True, 0.5)
    assert torch.equal(r, want[0]) and torch.equal(h, want[1])
    # the dense expert in 64 bits from the int8 rows: gate and up within 3 2^-24, SwiGLU (16 + 8 |g|) 2^-24,
    # half a bf16 step for act
    sf = lambda p: (p[1][:, 0] if p[1].dim() == 2 else p[1]).double()
    # (the sums of whole numbers first: they are exact in 64 bits)
    product = lambda a, b: (a[0].double() @ b[0].double().t().contiguous()) * sf(a)[:, None] * sf(b)
    gu = product(rows, shared[0])
    ga, up = gu[:, :SHARED].clamp(max=10), gu[:, SHARED:].clamp(-10, 10)
    ref = ga * torch.sigmoid(ga) * up
    assert bool(((act.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + (16 + 8 * ga.abs()) * U) + 1e-36).all())
    ref = product(rows2, shared[1])
    total = routed.double() + ref
    assert bool(((y.double() - total).abs() <= total.abs() * 2.0 ** -8 + 4 * U * (ref.abs() + routed.double().abs()) * 1.01).all())
    # the router's balance from the buffer that the block ran on
    loss, counts = dgm.router_balance_loss(logits, idx, z_coef=0.01)
    assert torch.equal(counts, stats)
    p = torch.softmax(logits.double(), 1)
    want_loss = float((E * counts.double() / (tokens * TOPK) * p.mean(0)).sum() + 0.01 * torch.logsumexp(logits.double(), 1).square().mean())
    assert abs(float(loss) - want_loss) <= 300 * U * want_loss


def test_without_the_options_and_in_a_graph():
    need_gpu()
    dgm, l1, l2, shared, b, w, rnd = setup()
    x = rnd(20, H)
    r, h = dgm.mega_moe_block(x, w["norm"], w["router"], l1, l2, b)
    _, h1 = dgm.rms_norm_residual(x, pre_weight=w["norm"])
    y = torch.empty_like(h1)
    dgm.mxfp4_mega_moe_from_bf16(y, h1, w["router"], l1, l2, b)
    assert h is None and torch.equal(r, dgm.rms_norm_residual(y, x)[0])
    run = lambda: dgm.mega_moe_block(x, w["norm"], w["router"], l1, l2, b, residual=x, shared_expert=shared,
                                     post_weight=w["post"], next_weight=w["next"])
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
        assert all(torch.equal(a, c) for a, c in zip(held, eager)), i


def test_block_refusals():
    need_gpu()
    dgm, l1, l2, shared, b, w, rnd = setup()
    x = rnd(4, H)
    call = lambda x=x, **kw: dgm.mega_moe_block(x, w["norm"], w["router"], l1, l2, b, **kw)
    with pytest.raises(TypeError, match="x must be bf16"):
        call(x.float())
    with pytest.raises(TypeError, match="x must be bf16"):
        call(rnd(4, H + 8))
    with pytest.raises(ValueError, match="shared_expert"):
        call(shared_expert=(shared[0], (shared[1][0][:, :128].contiguous(), shared[1][1])))
    with pytest.raises(RuntimeError, match="no gradient"):
        call(x.clone().requires_grad_())
