"""router_balance_loss where scores leave the middle of their range."""
import pytest
import torch

from tests.gpu_common import need_gpu
from tests.test_gpu_balance import U, check, close, formula, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [40, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_the_lowest_value(T, dtype):
    """Routed rows whose logits all are the type's lowest value: every expert alike, and without a z loss their
    logsumexp^2, beyond fp32, adds nothing."""
    need_gpu()
    logits, idx = make(T, 24, 2, dtype, seed=T)
    logits[3:6] = torch.finfo(dtype).min
    idx[3:6, 0] = torch.arange(3, device="cuda")
    for cuts in ([0, T], [0, 4, T]):
        loss, counts, d = run(logits, idx, cuts, 1.0, 0.0, "softmax")
        # (the same probabilities from logits of zero, whose formula has no sum that loses the logarithm)
        even = logits.clone()
        even[3:6] = 0
        want, wc, wg, wm = formula(even, idx, cuts, 1.0, 0.0, "softmax")
        assert torch.equal(counts.long().cpu(), wc) and abs(float(loss.detach()) - want) <= 300 * U * abs(want)
        close(d, wg, wm)


@pytest.mark.parametrize("T", [40, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_large_sigmoid_scores(T, dtype):
    """Logits up to 30: the factor 1 - sigmoid(l) = sigmoid(-l) relative to itself, (6 + |l|) 2^-24 more than the
    170 of the other factors."""
    need_gpu()
    logits, idx = make(T, 72, 4, dtype, seed=T + 1)
    logits = (logits.float() + torch.linspace(-20, 22, T, device="cuda")[:, None]).clamp(-30, 30).to(dtype)
    _, counts, d = run(logits, idx, [0, T], 1.0, 0.0, "sigmoid")
    l = logits.double().cpu()
    sg, rest = torch.sigmoid(l), torch.sigmoid(-l)
    p = sg / sg.sum(1, keepdim=True)
    routed = ((idx >= 0) & (idx < 72)).any(1).cpu()
    f = 72 * counts.double().cpu() / counts.sum().cpu()
    dot = (p * f).sum(1, keepdim=True)
    c = routed[:, None] / routed.sum() * p * rest
    close(d, c * (f - dot), c * (f + dot), 210)


@pytest.mark.parametrize("T", [40, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_vanishing_sigmoid_scores(T, dtype):
    """Rows of logits from -250 to -50: each sigmoid may lie below the least fp32 number, their shares do not."""
    need_gpu()
    logits, idx = make(T, 48, 4, dtype, seed=T + 2)
    logits = (logits.float().clamp(-12, 12) - torch.linspace(0, 238, T, device="cuda")[:, None]).to(dtype)
    check(logits, idx, [0, T], 1.0, 0.0, "sigmoid")
    check(logits, idx, [0, 11, 30, T], 1.0, 0.0, "sigmoid", g=-2.0)


@pytest.mark.parametrize("T", [40, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_sigmoid_rows_at_the_lowest_value(T, dtype):
    """Rows of the type's lowest value alone, or with masked experts beside it: the others share alike, and 1 - sigmoid
    is 1."""
    need_gpu()
    E = 24
    logits, idx = make(T, E, 2, dtype, seed=T)
    logits[3:6] = torch.finfo(dtype).min
    logits[5, 10:] = float("-inf")
    idx[3:6, 0] = torch.arange(3, device="cuda")
    loss, counts, d = run(logits, idx, [0, T], 1.0, 0.0, "sigmoid")
    l = logits.double().cpu()
    p, rest = torch.sigmoid(l), torch.sigmoid(-l)
    p[3:5], p[5] = 1.0, (torch.arange(E) < 10).double()
    p = p / p.sum(1, keepdim=True)
    routed = ((idx >= 0) & (idx < E)).any(1).cpu()
    f = E * counts.double().cpu() / counts.sum().cpu()
    want = float((f * p[routed].mean(0)).sum())
    assert abs(float(loss.detach()) - want) <= 300 * U * want
    dot = (p * f).sum(1, keepdim=True)
    c = routed[:, None] / routed.sum() * p * rest
    close(d, c * (f - dot), c * (f + dot), 210)
