"""Layer norm's largest rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_backward_of_the_widest_rows(gpu):
    """2^28 - 1 columns: the columns' sums of 2^22 workgroups."""
    import tinygnn_amd as tg
    cols = 2 ** 28 - 1
    x = torch.zeros(2, cols, dtype=torch.bfloat16, device="cuda")
    dy = torch.ones_like(x)
    dy[1, ::3] = -2
    x[0, -1] = 1
    y, mean, rstd = tg.layer_norm(x, with_stats=True)
    dx, dgamma, dbeta = tg.layer_norm_backward(dy, x, mean, rstd)
    want = dy.sum(0, dtype=torch.float32).to(x.dtype)
    assert torch.equal(dbeta, want)
    # xh is about 0 but in the last column, where it is rstd = 316 of the first row
    assert float(dgamma[:-1].abs().max()) < 1e-4
    assert abs(float(dgamma[-1]) - 316.2) < 1.3     # half a step of bf16 beside it
    assert torch.isfinite(dx).all() and torch.isfinite(y).all()
