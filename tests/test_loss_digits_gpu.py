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


@pytest.mark.parametrize("rows,classes", [(500, 2), (500, 7), (500, 41), (500, 53), (9000, 64),
                                          (9, 65), (700, 201), (40, 256)])
def test_the_same_distribution(gpu, rows, classes):
    """A teacher of all classes' logits, all equal: both logarithms are those of the same
    whole number, and every place's difference is 0."""
    import tinygnn_amd as tg
    x = torch.full((rows, classes), 0.75, device="cuda")
    ids = torch.arange(classes, device="cuda").to(I32).repeat(rows, 1)
    teacher = torch.full((rows, classes), -2.0, device="cuda")
    for temperature in (1.0, 3.0):
        loss = tg.distill(x, teacher, ids, temperature=temperature)
        assert not loss.any(), loss.abs().max()
        loss, d = tg.distill(x, teacher, ids, temperature=temperature,
                             dloss=torch.ones(rows, device="cuda"))
        assert not loss.any()
        # (p, q and their products by 1 / T: a few roundings of 1 / classes)
        within(d, torch.zeros_like(d), 10 * U / classes, "dlogits")


def test_loss_of_random_rows(gpu):
    """Losses of 41 classes in the 2-norm: no more than half as far again from 64
    bits as place by place in float32."""
    import head_cases as hc
    import tinygnn_amd as tg
    from expert_cases import gen, randn
    g, rows, classes, k = gen(3), 20_000, 41, 8
    x = randn(g, (rows, classes), torch.float32, 2.0)
    teacher, ids = torch.topk(x + 0.7 * randn(g, (rows, classes), torch.float32), k, 1)
    ids = ids.to(I32)
    want, _ = hc.distill(hc.Row(x, 2.0), teacher, ids, 2.0)
    z = (x - x.max(1, keepdim=True)[0]) * 0.5
    t = (teacher - teacher.max(1, keepdim=True)[0]) * 0.5
    q, log_q = torch.softmax(t, 1), torch.log_softmax(t, 1)
    plain = (q * (log_q - torch.gather(torch.log_softmax(z, 1), 1, ids.long()))).sum(1)
    off = [(v.double() - want).norm() for v in (plain, tg.distill(x, teacher, ids, temperature=2.0))]
    assert off[1] <= 1.5 * off[0], off
