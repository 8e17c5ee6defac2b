"""Routing, its plan, its backward pass and the join of the experts' results,
on the GPU against 64 bits.

Tolerances (u = 2^-24): exp's argument x - top is off by u |x - top|, exp and
the sum of up to 1,024 (16 a lane, then a tree) by 24 u, the quotient by u.
The join adds k terms in a chain: (k + 1) u; the dots add cols / 64 a lane."""
import pytest
import torch

from expert_cases import DTYPES, U, gen, half_step, least, padded, randn, within

pytestmark = pytest.mark.gpu


def reference(logits, k, renorm):
    """weights, experts, p by repeated search: the lowest index of the largest."""
    x = logits.double()
    t, e = x.shape
    left = torch.where(torch.isnan(x), -float("inf"), x)
    at = torch.arange(e, device=x.device)
    experts = []
    for _ in range(k):
        best = left.max(1, keepdim=True)[0]
        first = torch.where(left == best, at, e).min(1)[0]
        experts.append(torch.where(best[:, 0] > -float("inf"), first, -1))
        left[torch.arange(t, device=x.device), first] = -float("inf")
    experts = torch.stack(experts, 1)
    top = torch.where(torch.isnan(x), -float("inf"), x).max(1, keepdim=True)[0]
    p = torch.where(x == -float("inf"), 0.0, torch.exp(x - top))
    total = p.sum(1, keepdim=True)
    p = torch.where(total == 0, 0.0, p / total)
    bad = torch.isnan(p).any(1, keepdim=True)
    w = torch.where(experts >= 0, torch.gather(p, 1, experts.clamp_min(0)), 0.0)
    if renorm:
        part = w.sum(1, keepdim=True)
        w = torch.where(part == 0, 0.0, w / part)
    w = torch.where(bad, float("nan"), w)
    spread = torch.where(p > 0, (x - top).abs(), 0.0).nan_to_num().max(1, keepdim=True)[0]
    return w, experts.int(), p, (spread + 26) * U


def check_plan(plan, experts, n):
    """The plan from the experts, by a stable sort on the host."""
    flat = experts.reshape(-1).cpu()
    k = experts.shape[1] if experts.dim() == 2 else 1
    ids = torch.where((flat >= 0) & (flat < n), flat, n).long()
    order = torch.sort(ids, stable=True)[1]
    kept = int((ids < n).sum())
    offsets = torch.zeros(n + 1, dtype=torch.int64)
    offsets[1:] = torch.bincount(ids, minlength=n + 1)[:n].cumsum(0)
    rows = torch.full_like(order, -1)
    rows[:kept] = order[:kept] // k
    position = torch.full_like(order, -1)
    position[order[:kept]] = torch.arange(kept)
    assert torch.equal(plan.offsets.cpu().long(), offsets)
    assert torch.equal(plan.rows.cpu().long(), rows)
    assert torch.equal(plan.position.reshape(-1).cpu().long(), position)


def backward_reference(dw, w, experts, p, renorm):
    dw = torch.where(experts >= 0, dw.double(), 0.0)
    t, e = p.shape
    inner = (dw * torch.where(experts >= 0, w, 0.0)).sum(1, keepdim=True)
    size = (dw * w).abs().sum(1, keepdim=True)
    hit = torch.zeros(t, e + 1, dtype=torch.float64, device=p.device)
    at = torch.where(experts >= 0, experts, e).long()
    if renorm:
        return (hit.scatter(1, at, w * (dw - inner))[:, :e],
                hit.scatter(1, at, w * (dw.abs() + size))[:, :e])
    g = hit.scatter(1, at, dw)[:, :e]
    return p * (g - inner), p * (g.abs() + size)


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 4, 4), (8, 64, 2), (5, 65, 3),
                                              (256, 128, 8), (257, 100, 8), (300, 16, 16),
                                              (100, 24, 24), (77, 250, 32), (1000, 256, 5),
                                              (64, 257, 9), (700, 1000, 32), (70, 1024, 1),
                                              (20000, 60, 6), (70001, 9, 1)])
def test_route(gpu, tokens, experts, k, dtype, renorm):
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(tokens + 7 * experts + k)
    x = padded(randn(g, (tokens, experts), dt, 2.0), 3)
    w, ids, plan = tg.route(x, k, renormalize=renorm)
    want, eids, p, rel = reference(x, k, renorm)
    assert torch.equal(ids, eids)
    within(w, want, 2 * rel * want, "weights")
    check_plan(plan, ids, experts)
    dw = randn(g, (tokens, k), torch.float32)
    dl, size = backward_reference(dw, want, eids, p, renorm)
    got = tg.route_backward(dw, x, w, ids, renormalize=renorm)
    within(got, dl, (6 * rel + k * U) * size + half_step(dt) * dl.abs() + least(dt), "dlogits")


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("tokens", [40, 5000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_route_masks(gpu, dtype, tokens, renorm):
    """Masked experts, rows with none left, the type's lowest value, ties, NaN
    and +inf."""
    import tinygnn_amd as tg
    dt, g, e, k = DTYPES[dtype], gen(3), 48, 4
    x = randn(g, (tokens, e), dt)
    x[torch.rand((tokens, e), generator=g, device="cuda") < 0.4] = -float("inf")
    x[0::8] = -float("inf")                       # nothing left
    x[1::8, 2:] = -float("inf")                   # two left
    x[2::8] = torch.finfo(dt).min                 # the lowest value: an ordinary tie
    x[3::8, 1:] = torch.finfo(dt).min
    x[4::8] = torch.round(x[4::8].float()).to(dt)  # ties
    x[5, 7], x[13, 0], x[13, 3] = float("nan"), float("inf"), float("nan")
    x[6, 40] = float("inf")
    x[21] = float("nan")
    w, ids, plan = tg.route(x, k, renormalize=renorm)
    want, eids, p, rel = reference(x, k, renorm)
    assert torch.equal(ids, eids)
    assert torch.equal(torch.isnan(w), torch.isnan(want))
    within(w, want, 2 * rel * want.abs(), "weights")
    check_plan(plan, ids, e)
    assert bool((ids[0] == -1).all()) and bool((w[0] == 0).all())
    left = torch.isfinite(x[1]).nonzero().flatten().tolist()   # of the two, or none
    assert sorted(i for i in ids[1].tolist() if i >= 0) == left
    assert ids[1, len(left):].tolist() == [-1] * (k - len(left))
    assert ids[2].tolist() == [0, 1, 2, 3]
    dw = randn(g, (tokens, k), torch.float32)
    dw[1, 2] = float("nan")                       # of no expert: not used
    got = tg.route_backward(dw, x, w, ids, renormalize=renorm)
    ok = ~torch.isnan(want).any(1)
    dl, size = backward_reference(dw, want, eids, p, renorm)
    within(got[ok], dl[ok], ((6 * rel + k * U) * size + half_step(dt) * dl.abs() + least(dt))[ok])
    assert not got[0].any()


def test_route_without_a_plan(gpu):
    """The C entry with no plan asked for; keyword arguments of the front end."""
    import tinygnn_amd as tg
    x = randn(gen(2), (300, 20), torch.float32)
    w, ids, _ = tg.route(logits=x, k=3)
    w2, ids2 = torch.empty_like(w), torch.empty_like(ids)
    tg.lib.check(tg.lib.tg_route(300, 20, 3, tg.TYPE_F32, x.data_ptr(), 20, 0, w2.data_ptr(),
                                 ids2.data_ptr(), None, None, None, None, 0,
                                 tg.stream_handle()))
    assert torch.equal(w, w2) and torch.equal(ids, ids2)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 8192, 8193, 100_003, 1_200_000])
@pytest.mark.parametrize("groups", [1, 2, 7, 64, 1000, 1024])
def test_plan(gpu, n, groups):
    """Node types: some ids outside the groups, some groups empty."""
    import tinygnn_amd as tg
    g = gen(n + groups)
    ids = torch.randint(-1, groups + 2, (n,), generator=g, device="cuda", dtype=torch.int32)
    ids[ids == groups // 2] = 0
    ids[ids == groups + 1] = 2 ** 31 - 1
    plan = tg.route_plan(ids, groups)
    check_plan(plan, ids, groups)
    if n % 4 == 0:
        check_plan(tg.route_plan(ids.view(-1, 4), groups), ids.view(-1, 4), groups)


def test_plan_of_nothing(gpu):
    import tinygnn_amd as tg
    plan = tg.route_plan(torch.empty(0, dtype=torch.int32, device="cuda"), 5)
    assert plan.offsets.tolist() == [0] * 6 and plan.rows.numel() == 0
    w, ids, plan = tg.route(torch.empty(0, 6, device="cuda"), 2)
    assert w.shape == ids.shape == (0, 2) and plan.offsets.tolist() == [0] * 7
    assert tg.route_backward(w, torch.empty(0, 6, device="cuda"), w, ids).shape == (0, 6)


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,k,cols", [(1, 1, 1), (3, 2, 8), (5, 9, 511), (300, 4, 2048),
                                           (64, 32, 257), (9, 3, 5000), (2001, 1, 41),
                                           (40, 8, 1024), (17, 13, 1500)])
def test_combine(gpu, tokens, k, cols, dtype, weighted):
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(tokens + k + cols)
    rows = tokens * k + 5
    y = padded(randn(g, (rows, cols), dt), 1)
    pos = torch.randperm(rows, generator=g, device="cuda")[:tokens * k].view(tokens, k).int()
    pos[torch.rand((tokens, k), generator=g, device="cuda") < 0.2] = -1
    pos[0] = torch.where(pos[0] >= 0, pos[0], rows + 3)    # outside: nothing
    w = randn(g, (tokens, k), torch.float32) if weighted else None
    dout = padded(randn(g, (tokens, cols), dt), 2)
    live = (pos >= 0) & (pos < rows)
    at = torch.where(live, pos, 0).long()
    f = (torch.ones(tokens, k, dtype=torch.float64, device="cuda") if w is None else w.double())
    f = torch.where(live, f, 0.0)
    mine = torch.where(live[:, :, None], y.double()[at], 0.0)
    want, size = (mine * f[:, :, None]).sum(1), (mine * f[:, :, None]).abs().sum(1)
    got = tg.route_combine(y, pos, w)
    within(got, want, (k + 1) * U * size + half_step(dt) * want.abs() + least(dt), "out")
    before = randn(g, (rows, cols), dt)
    dy = before.clone()
    got_dy, dw = tg.route_combine_backward(dout, y, pos, w, out=dy)
    assert got_dy is dy
    want = before.double().clone()
    want[at[live]] = (f[:, :, None] * dout.double()[:, None])[live]
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    named[at[live]] = True
    assert torch.equal(dy[~named], before[~named])
    within(dy, want, (U + half_step(dt)) * want.abs() + least(dt), "dy")
    dots = (mine * dout.double()[:, None]).sum(2)
    size = (mine * dout.double()[:, None]).abs().sum(2)
    within(dw, dots, (cols / 64 + 12) * U * size, "dweights")


def test_combine_leaves_nan_of_others(gpu):
    """Rows that no position names may hold anything."""
    import tinygnn_amd as tg
    y = torch.full((4, 300), float("nan"), device="cuda")
    y[2] = 1.5
    pos = torch.tensor([[2, -1], [-1, -1], [7, -5]], dtype=torch.int32, device="cuda")
    out = tg.route_combine(y, pos, torch.full((3, 2), 2.0, device="cuda"))
    assert bool((out[0] == 3).all()) and not out[1:].any()
