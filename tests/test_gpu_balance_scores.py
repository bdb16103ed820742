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
