"""Log probabilities, the entropy, the top classes, distillation, and their
gradients, on the GPU against 64 bits (bounds: head_cases.py)."""
import pytest
import torch

import head_cases as hc
from expert_cases import DTYPES, gen, padded, randn, within

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
I32 = torch.int32

SIZES = [(1, 1), (3, 2), (700, 7), (65, 41), (64, 47), (1, 41), (7, 64), (9, 65), (200, 100),
         (33, 257), (5, 511), (3, 1000), (4, 1025), (2, 2048), (3, 2049), (2, 4097), (2, 8200),
         (300, 5000), (1, 16384), (2, 32000), (1, 32769), (3, 65537), (1, 131072), (2, 131079),
         (1, 200003), (1, 1100001), (20011, 41), (600, 9001), (1030, 3000), (1030, 12000),
         (1030, 30000), (1030, 60000)]


def make(rows, classes, dt, seed):
    g = gen(seed)
    x = torch.randn((rows, classes), generator=g, device="cuda")
    x = x * (0.5 + 3 * torch.rand((rows, 1), generator=g, device="cuda"))
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    if classes > 4:
        x[torch.rand((rows, classes), generator=g, device="cuda") < 0.05] = -INF
        x[torch.arange(rows, device="cuda"), labels] = 1.5
    labels[3::7] = -1
    labels[5::11] = classes + 5
    return g, x.to(dt), labels.to(I32)


def check_log_probs(x, labels, top, temperature, dvalue=None, dentropy=None, out=None):
    import tinygnn_amd as tg
    dt = x.dtype
    row = hc.Row(x, temperature)
    r = tg.log_probs(x, labels, top=top, entropy=True, temperature=temperature)
    want, tol = hc.value(row, labels)
    within(hc.in_range(r.value, want, tol), want, tol, "value")
    ent = torch.where(row.nan, NAN, torch.where(row.empty, 0.0, row.entropy))
    within(r.entropy, ent, row.entropy_tol, "entropy")
    if top:
        ids = hc.top(x, top)
        assert torch.equal(r.top_ids, ids.to(I32))
        at = ids.clamp_min(0)
        v = torch.where(ids >= 0, torch.gather(row.logp, 1, at), -INF)
        v = torch.where(row.nan[:, None] & (ids >= 0), NAN, v)
        tol = torch.gather(row.at, 1, at)
        within(hc.in_range(r.top_values, v, tol), v, tol, "top values")
    else:
        assert r.top_ids is None and r.top_values is None
    for dv, dh in ((dvalue, None), (None, dentropy), (dvalue, dentropy)):
        if dv is None and dh is None:
            continue
        d, tol = hc.backward(row, labels, dv, dh, temperature)
        got = tg.log_probs_backward(dv, x, labels if dv is not None else None, r, dentropy=dh)
        within(got, d, hc.rounded(torch.nan_to_num(d), tol, dt), "dlogits")
    return r


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", SIZES)
def test_log_probs(gpu, rows, classes, dtype):
    g, x, labels = make(rows, classes, DTYPES[dtype], rows + classes)
    x = padded(x, 3)
    dvalue, dentropy = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    for top, temperature in ((0, 1.0), (min(5, classes), 0.7), (min(20, classes), 1.0),
                             (min(64, classes), 3.0)):
        check_log_probs(x, labels, top, temperature, dvalue, dentropy)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", [(1, 20_001), (1, 40_003), (127, 20_003), (127, 40_005),
                                          (128, 48_001), (130, 151_001), (1023, 95_005),
                                          (1024, 95_001)])
def test_rows_whole_and_cut(gpu, rows, classes, dtype):
    """At both sides of where rows are cut."""
    g, x, labels = make(rows, classes, DTYPES[dtype], rows + classes)
    dvalue, dentropy = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    for top in (0, 20):
        check_log_probs(x, labels, top, 0.9, dvalue, dentropy)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", SIZES)
def test_distill(gpu, rows, classes, dtype):
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    g, x, _ = make(rows, classes, dt, rows + classes + 1)
    x = padded(x, 3)
    dloss = torch.randn(rows, generator=g, device="cuda")
    dloss[2::5] = 0
    for k, temperature, kind in ((1, 1.0, dt), (8, 2.0, torch.float32), (33, 0.7, dt),
                                 (256, 1.0, torch.bfloat16)):
        if k > 33 and rows * classes > 2_000_000:
            continue   # the oracle's time
        ids = torch.randint(-1, classes + 1, (rows, k), generator=g, device="cuda").to(I32)
        # the same class several times, and (mostly) unmasked ones
        if k > 8:
            ids[:, 5] = ids[:, 2]
            ids[:, 6] = ids[:, 2]
        teacher = randn(g, (rows, k), kind, 2.0)
        row = hc.Row(x, temperature)
        loss, tol, d, dt_ = hc.distill(row, teacher, ids, temperature, dloss)
        within(tg.distill(x, teacher, ids, temperature=temperature), loss, tol, "loss")
        got, grad = tg.distill(x, teacher, ids, temperature=temperature, dloss=dloss)
        within(got, loss, tol, "loss with gradient")
        within(grad, d, hc.rounded(torch.nan_to_num(d), dt_, dt), "dlogits")


MASK_SIZES = [(60, 48), (60, 300), (40, 3000), (40, 20000), (40, 70000), (600, 40)]


def masked(rows, classes, dt):
    """Every kind of row: all masked, one class left, the type's lowest value,
    ties, NaN, infinities, far apart values."""
    g, x, labels = make(rows, classes, dt, 3)
    low, high = torch.finfo(dt).min, torch.finfo(dt).max
    x[0::10] = -INF
    x[1::10] = -INF
    x[1::10, 3] = 2.0
    x[2::10] = low
    x[3::10, 5:] = low
    x[4::10] = torch.round(x[4::10].float().nan_to_num(0, 0, 0)).to(dt)
    x[5::10] = 0
    x[6::20, 7] = NAN
    x[16::20, 9] = INF
    x[7::20] = NAN
    x[17::20, 1:] = INF
    x[8::10, 0], x[8::10, 1] = high, low
    x[9::10, 2:] = -INF
    return g, x, labels


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", MASK_SIZES)
def test_masks(gpu, rows, classes, dtype):
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    g, x, labels = masked(rows, classes, dt)
    dvalue = torch.randn(rows, generator=g, device="cuda")
    dvalue[26::30] = 0           # a NaN row of no gradient
    dvalue[labels < 0] = NAN     # not used
    dentropy = torch.randn(rows, generator=g, device="cuda")
    dentropy[::2] = 0
    for top in (0, 4, 40):
        check_log_probs(x, labels, top, 1.0, dvalue, dentropy)
    # distillation: places of masked classes, none, NaN, -inf
    k = 6
    ids = torch.randint(0, classes, (rows, k), generator=g, device="cuda").to(I32)
    ids[::4, 2] = -1
    ids[5::9] = -1
    teacher = randn(g, (rows, k), torch.float32)
    teacher[::3, 4] = -INF
    teacher[12::13] = -INF
    teacher[14, 1], teacher[25, 0] = NAN, INF
    row = hc.Row(x, 1.0)
    dloss = torch.randn(rows, generator=g, device="cuda")
    dloss[36] = 0
    loss, tol, d, dtol = hc.distill(row, teacher, ids, 1.0, dloss)
    got, grad = tg.distill(x, teacher, ids, dloss=dloss)
    within(hc.in_range(got, loss, tol), loss, tol, "loss")
    within(grad, d, hc.rounded(torch.nan_to_num(d), dtol, dt), "dlogits")


@pytest.mark.parametrize("classes", [5, 300, 5000, 70000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_falling_and_equal_rows(gpu, classes, dtype):
    """Rows in rising and falling order, and of one value: every top place
    comes from one part of the row."""
    dt = DTYPES[dtype]
    ramp = torch.linspace(-4, 4, classes, device="cuda")
    rows = [ramp, -ramp, 0 * ramp, ramp.abs(), -ramp.abs()]
    # large values on few of the threads that may share a row
    at = torch.arange(classes, device="cuda")
    for period in (8 * 16, 8 * 64, 8 * 256, 8 * 1024, 4 * 64, 4 * 1024):
        rows.append((at % period).float() / period + (at % 7) / 70)
        rows.append((at % period >= period // 2).float() + ramp / 10)
    x = torch.stack(rows).to(dt)
    labels = torch.arange(len(rows), device="cuda").to(I32) % classes
    many = x.repeat(1 + 600 // len(rows), 1)   # as many rows, too
    for top in (2, 31, 64):
        check_log_probs(x, labels, min(top, classes), 1.0)
        check_log_probs(many, labels.repeat(1 + 600 // len(rows)), min(top, classes), 1.0)


@pytest.mark.parametrize("rows,classes", [(50, 30), (30, 700), (9, 9000), (2, 150000)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_in_place(gpu, rows, classes, dtype):
    """The gradient over the logits; what lies between the rows stays."""
    import tinygnn_amd as tg
    g, x, labels = make(rows, classes, DTYPES[dtype], 9)
    dvalue = torch.randn(rows, generator=g, device="cuda")
    r = tg.log_probs(x, labels, entropy=True)
    want = tg.log_probs_backward(dvalue, x, labels, r, dentropy=dvalue)
    wide = padded(x, 5, fill=7.0)
    got = tg.log_probs_backward(dvalue, wide, labels, r, dentropy=dvalue, out=wide)
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got, want)
    assert bool((wide.as_strided((rows, 5), wide.stride(), classes) == 7.0).all())
    ids = torch.randint(0, classes, (rows, 9), generator=g, device="cuda").to(I32)
    teacher = randn(g, (rows, 9), torch.float32)
    loss, want = tg.distill(x, teacher, ids, dloss=dvalue)
    wide = padded(x, 5, fill=7.0)
    loss2, got = tg.distill(wide, teacher, ids, dloss=dvalue, out=wide)
    assert torch.equal(got, want) and torch.equal(loss, loss2)
    assert bool((wide.as_strided((rows, 5), wide.stride(), classes) == 7.0).all())


def test_empty_and_absent(gpu):
    """No rows; no labels; a teacher's file from log_probs' own top classes."""
    import tinygnn_amd as tg
    x = torch.zeros(0, 9, device="cuda")
    none = torch.zeros(0, dtype=I32, device="cuda")
    r = tg.log_probs(x, none, top=2, entropy=True)
    assert r.value.shape == (0,) and r.top_ids.shape == (0, 2)
    assert tg.log_probs_backward(r.value, x, none, r).shape == (0, 9)
    loss, d = tg.distill(x, torch.zeros(0, 3, device="cuda"), none.view(0, 3), dloss=r.value)
    assert loss.shape == (0,) and d.shape == (0, 9)
    g, x, _ = make(50, 500, torch.float32, 4)
    t = tg.log_probs(x, top=500 // 8)
    assert t.value is None and t.entropy is None
    # the teacher is the student: the divergence is the log of the mass kept
    kept = torch.exp(t.top_values.double()).sum(1)
    row = hc.Row(x, 1.0)
    loss, tol = hc.distill(row, t.top_values, t.top_ids, 1.0)
    got = tg.distill(x, t.top_values, t.top_ids)
    within(got, loss, tol, "loss")
    # (its own bound: that of the values, twice)
    within(got, -torch.log(kept), tol + 4 * row.at.max(1)[0], "divergence")


def test_gradients_by_differences(gpu):
    """Along each gradient's own direction, central differences of the forward
    form in 64 bits: steps of 1e-4 leave a third derivative of size 1 times 1e-8,
    and roundings of 2^-53 * 100 / 1e-4 < 1e-9."""
    import tinygnn_amd as tg
    g, x, labels = make(40, 200, torch.float32, 6)
    x = x.nan_to_num(0, 0, -3.0)
    labels = labels.clamp(0, 199)
    a, b = (torch.randn(40, generator=g, device="cuda") for _ in range(2))
    t, step = 1.3, 1e-4
    r = tg.log_probs(x, labels, entropy=True, temperature=t)
    teacher = randn(g, (40, 7), torch.float32)
    ids = torch.randint(0, 200, (40, 7), generator=g, device="cuda").to(I32)

    def logp(v):
        row = hc.Row(v, t)
        return (hc.value(row, labels)[0] * a.double() + row.entropy * b.double()).sum()

    def div(v):
        return (hc.distill(hc.Row(v, t), teacher, ids, t)[0] * a.double()).sum()

    for grad, loss in ((tg.log_probs_backward(a, x, labels, r, dentropy=b), logp),
                       (tg.distill(x, teacher, ids, temperature=t, dloss=a)[1], div)):
        d = grad.double() / grad.double().norm()
        want = (loss(x.double() + step * d) - loss(x.double() - step * d)) / (2 * step)
        got = grad.double().norm()
        assert abs(got - want) <= 1e-6 + 1e-5 * abs(want), (got, want)
