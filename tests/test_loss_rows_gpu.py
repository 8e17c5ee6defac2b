"""How many threads take a row of the losses, by the kernel that ran, on either side
of the rules that choose: ties, masks, NaN and infinities among the rows; against 64
bits (bounds: head_cases.py)."""
import re

import pytest
import torch

import head_cases as hc
from expert_cases import DTYPES, randn, within
from test_losses_gpu import check_log_probs, make, masked
from test_tile_shapes_gpu import kernels

pytestmark = pytest.mark.gpu
I32 = torch.int32
NAN, INF = float("nan"), float("inf")


def threads(names):
    """Threads of a row (1: a thread takes one), or None where the profiler sees no
    kernel."""
    if not any("_kernel" in n for n in names):
        return None
    if any("tiny_kernel" in n for n in names):
        return 1
    return int(re.search(r"row_kernel(?:<[^,]*, |I.*?Li)(\d+)", " ".join(names))[1])


def log_probs(x, labels, top, temperature, want):
    import tinygnn_amd as tg
    g = torch.Generator(device="cuda").manual_seed(len(x))
    dvalue, dentropy = (torch.randn(len(x), generator=g, device="cuda") for _ in range(2))
    dentropy[::3] = 0
    check_log_probs(x, labels, top, temperature, dvalue, dentropy)
    for entropy in (False, True):
        _, names = kernels(lambda: tg.log_probs(x, labels, top=top, entropy=entropy))
        assert threads(names) in (None, want), (names, want)


def chunk(dt):
    return 16 // dt.itemsize


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [513, 1030])
@pytest.mark.parametrize("classes", [65, 127, 255, 257, 470, 512, 513, 1000, 1024, 1025])
def test_rows_of_16_lanes(gpu, classes, rows, dtype):
    """Without top classes or with one: up to 128 chunks of 16 bytes; a wavefront for
    more, or for more top classes.  The last workgroup's rows are not all there."""
    dt = DTYPES[dtype]
    _, x, labels = masked(rows, classes, dt)
    want = 16 if classes <= 128 * chunk(dt) else 64
    for top, shape in ((0, want), (1, want), (2, 64)):
        log_probs(x, labels, top, 0.8, shape)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", [(20, 300), (20, 1025), (20, 20_003), (20, 131_079),
                                          (600, 5000), (300, 60_000), (200, 131_071)])
def test_the_likeliest_class(gpu, rows, classes, dtype):
    """One top class of whole and cut rows."""
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    _, x, labels = masked(rows, classes, dt)
    check_log_probs(x, labels, 1, 1.0, torch.ones(rows, device="cuda"))
    # the largest value in many places: the first, wherever that is
    last = torch.full((4, classes), 0.5, device="cuda").to(dt)
    at = [0, classes - 1, classes // 2, 1]
    for r, c in enumerate(at):
        last[r, :c] = -1.0
    r = tg.log_probs(last, top=1)
    assert r.top_ids[:, 0].tolist() == at


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("classes", [64, 65, 98, 127, 128, 129])
def test_rows_of_a_thread(gpu, classes, dtype):
    """Many rows: up to 128 classes with top classes or a teacher of up to 64 places,
    more than 64 KB of LDS at the most."""
    import tinygnn_amd as tg
    dt, rows = DTYPES[dtype], 8193
    _, x, labels = masked(rows, classes, dt)
    few = 1 if classes <= 128 else 16
    log_probs(x, labels, 1, 1.0, few)
    for top in (20, 64):
        log_probs(x, labels, top, 1.3, 1 if classes <= 128 else 64)
    log_probs(x, labels, 0, 1.0, 1 if classes <= 64 else 16)
    for k in (1, 8, 64, 65):
        one = 1 if classes <= 128 and k <= 64 else 64
        distill(x, k, one)


def distill(x, k, want):
    import tinygnn_amd as tg
    dt, (rows, classes) = x.dtype, x.shape
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.randint(-1, classes + 1, (rows, k), generator=g, device="cuda").to(I32)
    teacher = randn(g, (rows, k), dt, 2.0)
    ids[7::11] = -1
    teacher[3::17, 0] = -INF
    if k > 4:   # the same class several times
        ids[:, 4] = ids[:, 1]
        ids[::2, 3] = ids[::2, 1]
    dloss = torch.randn(rows, generator=g, device="cuda")
    dloss[4::9] = 0
    loss, tol, d, dtol = hc.distill(hc.Row(x, 1.5), teacher, ids, 1.5, dloss)
    (got, grad), names = kernels(lambda: tg.distill(x, teacher, ids, temperature=1.5, dloss=dloss))
    assert threads(names) in (None, want), (names, want)
    within(hc.in_range(got, loss, tol), loss, tol, "loss")
    within(grad, d, hc.rounded(torch.nan_to_num(d), dtol, dt), "dlogits")
    alone = tg.distill(x, teacher, ids, temperature=1.5)
    within(hc.in_range(alone, loss, tol), loss, tol, "loss alone")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,chunks,want", [(600, 65, 64), (600, 256, 64), (1031, 257, 64),
                                              (600, 1024, 64), (600, 1025, 256), (513, 4097, 1024),
                                              (9, 65, 256), (9, 1025, 1024), (9, 4999, 1024)])
def test_distill_by_rows(gpu, rows, chunks, want, dtype):
    """A wavefront up to 1,024 chunks of a row, then 256 and 1,024 threads; of few rows
    256 from 65 on; the last chunk of one value."""
    dt = DTYPES[dtype]
    _, x, _ = masked(rows, (chunks - 1) * chunk(dt) + 1, dt)
    for k in (3, 70):
        distill(x, k, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1.0, 3.0, 100.0, 1e4])
@pytest.mark.parametrize("rows,classes", [(9, 7), (9000, 70), (700, 300), (9, 700), (5, 70_000)])
def test_far_apart_logits(gpu, rows, classes, temperature, dtype):
    """The type's largest value and its lowest in one row: their difference lies past
    float32, over the temperature it may not."""
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    _, x, labels = make(rows, classes, dt, 4)
    x[:, 0], x[:, 1] = torch.finfo(dt).max, torch.finfo(dt).min
    x[1::2, 0] = 0.5 * torch.finfo(dt).max
    labels[:] = 1
    row = hc.Row(x, temperature)
    want, tol = hc.value(row, labels)
    r = tg.log_probs(x, labels, top=min(classes, 64), temperature=temperature)
    within(hc.in_range(r.value, want, tol), want, tol, "value")
    assert temperature == 1.0 or torch.isfinite(r.value).all()
    ids = hc.top(x, min(classes, 64))
    v = torch.where(ids >= 0, torch.gather(row.logp, 1, ids.clamp_min(0)), -INF)
    tol = torch.gather(row.at, 1, ids.clamp_min(0))
    within(hc.in_range(r.top_values, v, tol), v, tol, "top values")
    ids = torch.tensor([1, 0, 3], dtype=I32, device="cuda").repeat(rows, 1)
    x[:, 3] = 2.0
    teacher = torch.tensor([0.0, 1.0, 2.0], device="cuda").repeat(rows, 1)
    loss, tol = hc.distill(hc.Row(x, temperature), teacher, ids, temperature)
    got = tg.distill(x, teacher, ids, temperature=temperature)
    within(hc.in_range(got, loss, tol), loss, tol, "loss")
