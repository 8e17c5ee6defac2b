"""Digits of the losses' float32 gradients: rows of equal logits, whose exponentials
are 1 and whose sums are whole numbers, so that what is left are a few roundings."""
import pytest
import torch

from expert_cases import U, within

pytestmark = pytest.mark.gpu
I32 = torch.int32
# a thread, 16 lanes, a wavefront, a workgroup a row; cut rows
SIZES = [(500, 53), (9000, 112), (700, 201), (3, 717), (600, 717), (4, 7786), (600, 7786),
         (40, 15_013), (200, 49_970), (2, 130_051), (200, 130_051)]


@pytest.mark.parametrize("temperature", [1.0, 0.5])
@pytest.mark.parametrize("rows,classes", SIZES)
def test_distill(gpu, rows, classes, temperature):
    """dloss / T / classes: its products by 1 / T = 2 are exact; a quotient off by
    2.5 steps at most (5 u) and two products."""
    import tinygnn_amd as tg
    x = torch.full((rows, classes), 1.25, device="cuda")
    ids = torch.zeros(rows, 1, dtype=I32, device="cuda")
    dloss = 1 + torch.rand(rows, device="cuda")
    teacher = torch.zeros(rows, 1, device="cuda")
    _, d = tg.distill(x, teacher, ids, temperature=temperature, dloss=dloss)
    g = dloss.double()[:, None] / temperature
    want = (g / classes).expand(rows, classes).clone()
    want[:, 0] -= g[:, 0]
    within(d, want, 7 * U * want.abs(), "dlogits")


@pytest.mark.parametrize("rows,classes", SIZES)
def test_log_probs(gpu, rows, classes):
    """Against the sums' logarithm that the forward pass gives: an exponential off
    by one step (2 u), and two products."""
    import tinygnn_amd as tg
    x = torch.full((rows, classes), -3.5, device="cuda")
    labels = torch.zeros(rows, dtype=I32, device="cuda")
    dvalue = 1 + torch.rand(rows, device="cuda")
    r = tg.log_probs(x, labels)
    d = tg.log_probs_backward(dvalue, x, labels, r)
    g = dvalue.double()[:, None]
    want = -g * torch.exp(-r.stats[:, 1:].double()).expand(rows, classes)
    want = want.clone()
    want[:, 0] += g[:, 0]
    within(d, want, 5 * U * want.abs(), "dlogits")
