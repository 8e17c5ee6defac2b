"""Dense layers, log probabilities and distillation together: a network of dense
layers taught by another's top classes and by labels; on another stream; two at
once; captured into a graph and replayed; far offsets."""
import pytest
import torch

import head_cases as hc
from expert_cases import DTYPES, gen, randn, within

pytestmark = pytest.mark.gpu
T, D, H, C, K = 300, 40, 72, 50, 6
I32 = torch.int32


def inputs(dtype, seed=1):
    g = gen(seed)
    p = dict(x=randn(g, (T, D), dtype), w1=randn(g, (D, H), dtype, D ** -0.5),
             b1=randn(g, H, dtype, 0.1), w2=randn(g, (H, H), dtype, H ** -0.5),
             b2=randn(g, H, dtype, 0.1), w3=randn(g, (C, H), dtype, H ** -0.5))
    p["teacher"] = randn(g, (T, C), torch.float32, 2.0)
    labels = torch.randint(0, C, (T,), generator=g, device="cuda").to(I32)
    labels[5::9] = -1
    p["labels"] = labels
    p["dloss"] = torch.rand(T, generator=g, device="cuda")
    p["dvalue"] = -torch.rand(T, generator=g, device="cuda")
    p["dentropy"] = 0.1 * torch.rand(T, generator=g, device="cuda")
    return p


def step(tg, p, stream=None):
    """Two hidden layers, the second with a residual, and the classes; the
    teacher's places come from log_probs."""
    s = dict(stream=stream)
    taught = tg.log_probs(p["teacher"], top=K, **s)
    h1, pre1 = tg.linear(p["x"], p["w1"], bias=p["b1"], epilogue=tg.EPI_GELU, with_pre=True, **s)
    h2, pre2 = tg.linear(h1, p["w2"], bias=p["b2"], epilogue=tg.EPI_SILU, residual=h1,
                         with_pre=True, **s)
    z = tg.linear(h2, p["w3"], transpose=True, **s)
    loss, dz = tg.distill(z, taught.top_values, taught.top_ids, temperature=2.0, dloss=p["dloss"],
                          **s)
    r = tg.log_probs(z, p["labels"], entropy=True, **s)
    dz = dz + tg.log_probs_backward(p["dvalue"], z, p["labels"], r, dentropy=p["dentropy"], **s)
    dh2, dw3, _ = tg.linear_backward(dz, h2, p["w3"], transpose=True, **s)
    dh1, dw2, db2 = tg.linear_backward(dh2, h1, p["w2"], pre=pre2, epilogue=tg.EPI_SILU, bias=True,
                                       **s)
    dx, dw1, db1 = tg.linear_backward(dh1 + dh2, p["x"], p["w1"], pre=pre1, epilogue=tg.EPI_GELU,
                                      bias=True, **s)
    return dict(z=z, loss=loss, value=r.value, dx=dx, dw1=dw1, db1=db1, dw2=dw2, db2=db2, dw3=dw3,
                ids=taught.top_ids)


def reference(p):
    """The same in 64 bits by torch's differentiation."""
    q = {k: v.double().requires_grad_() if k in ("x", "w1", "b1", "w2", "b2", "w3") else v
         for k, v in p.items()}
    top = hc.top(p["teacher"], K)
    t = torch.gather(p["teacher"].double(), 1, top)
    teacher = torch.softmax(t / 2.0, 1)
    h1 = torch.nn.functional.gelu(q["x"] @ q["w1"] + q["b1"], approximate="tanh")
    h2 = h1 + torch.nn.functional.silu(h1 @ q["w2"] + q["b2"])
    z = h2 @ q["w3"].t()
    soft = torch.gather(torch.log_softmax(z / 2.0, 1), 1, top)
    loss = (teacher * (teacher.log() - soft)).sum(1)
    logp = torch.log_softmax(z, 1)
    given = p["labels"] >= 0
    value = torch.where(given, torch.gather(logp, 1, p["labels"].clamp_min(0).long()[:, None])[:, 0],
                        0.0)
    entropy = -(logp.exp() * logp).sum(1)
    total = ((loss * p["dloss"].double()).sum() + (value * p["dvalue"].double()).sum()
             + (entropy * p["dentropy"].double()).sum())
    names = ["x", "w1", "b1", "w2", "b2", "w3"]
    grads = torch.autograd.grad(total, [q[n] for n in names])
    out = dict(z=z.detach(), loss=loss.detach(), value=value.detach())
    out.update({"d" + n: g for n, g in zip(names, grads)})
    return out, top


@pytest.mark.parametrize("dtype,share", [(torch.float32, 2e-5), (torch.bfloat16, 6e-2)])
def test_step(gpu, dtype, share):
    """share: of the largest value of each result.  float32: sums of at most 300
    terms with 100 u each way through six products, 6 * 300 * 2^-24 = 1.1e-4 of
    their sizes in the worst case, a tenth of it for sums of random signs; bf16: a
    dozen roundings of 2^-9 one after another, forward and back, are 12 * 2^-9 =
    2.4e-2, and the softmax of logits of size 4 takes up to 4 times its own of the
    last three."""
    import tinygnn_amd as tg
    p = inputs(dtype)
    got, (want, top) = step(tg, p), reference(p)
    assert torch.equal(got["ids"], top.to(I32))
    for name, v in want.items():
        within(got[name], v, share * v.abs().max(), name)


def test_step_on_another_stream(gpu):
    """Inputs come from a long queue on the current stream; results of another one
    are read at once."""
    import tinygnn_amd as tg
    p = inputs(torch.float32)
    want = step(tg, p)
    late = {k: torch.zeros_like(v) for k, v in p.items()}
    big, side = torch.randn(4096, 4096, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        big = torch.mm(big, big)
    for k, v in p.items():
        late[k].copy_(v)
    got = step(tg, late, stream=side)
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_steps_on_two_streams(gpu):
    import tinygnn_amd as tg
    ps = [inputs(torch.bfloat16, seed) for seed in (3, 4)]
    want = [step(tg, p) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(tg, ps[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for name in w:
            assert torch.equal(g[name], w[name]), name


def test_two_captured_steps(gpu):
    """Two graphs of the same calls, replayed in turn on new inputs, eager calls in
    between; cut rows and contractions among them, which take workspaces."""
    import tinygnn_amd as tg

    def run(p):
        out = step(tg, p)
        r = tg.log_probs(p["long"], top=9, entropy=True)
        loss, d = tg.distill(p["long"], r.top_values, r.top_ids, dloss=p["dloss"][:2])
        dx, dw, db = tg.linear_backward(p["tall"][:, :24], p["tall"], p["narrow"], bias=True)
        out.update(top=r.top_ids, far=loss, dlong=d, cut=tg.linear(p["wide"], p["deep"]), dn=dw,
                   dt=dx, db=db)
        return out

    def fresh(seed):
        g, p = gen(seed), inputs(torch.float32, seed)
        p.update(long=randn(g, (2, 70_000), torch.float32, 2.0),
                 wide=randn(g, (40, 9000), torch.float32),
                 deep=randn(g, (9000, 30), torch.float32),
                 tall=randn(g, (20_000, 48), torch.float32),
                 narrow=randn(g, (48, 24), torch.float32))
        return p

    statics, graphs, outs = [fresh(0), fresh(0)], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(statics[0])
    torch.cuda.current_stream().wait_stream(side)
    for p in statics:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(p))
        graphs.append(graph)
    for seed in (1, 2, 3, 4):
        new = [fresh(seed), fresh(seed + 10)]
        want = [run(p) for p in new]
        for p, v in zip(statics, new):
            for k in p:
                p[k].copy_(v[k])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for name in w:
                assert torch.equal(o[name], w[name]), (seed, name)


def test_capture_without_workspace_is_refused(gpu):
    import tinygnn_amd as tg
    x, y = torch.randn(40, 9000, device="cuda"), torch.empty(40, 30, device="cuda")
    w, loss = torch.randn(9000, 30, device="cuda"), torch.empty(1, device="cuda")
    z, t = torch.randn(1, 70_000, device="cuda"), torch.zeros(1, 3, device="cuda")
    ids = torch.zeros(1, 3, dtype=I32, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.capture_begin(capture_error_mode="relaxed")
        rcs = [tg.lib.tg_linear(40, 9000, 30, 0, x.data_ptr(), 9000, w.data_ptr(), 30, 0, None, 0,
                                None, 0, y.data_ptr(), 30, None, 0, None, 0, int(side.cuda_stream)),
               tg.lib.tg_distill(1, 70_000, 3, 0, z.data_ptr(), 70_000, 0, t.data_ptr(),
                                 ids.data_ptr(), 1.0, loss.data_ptr(), None, None, 0, None, 0,
                                 int(side.cuda_stream))]
        graph.capture_end()
    assert rcs == [1, 1] and b"being captured" in tg.lib.tg_last_error()


def test_without_a_workspace(gpu):
    """The library's own temporaries: the same bits."""
    import tinygnn_amd as tg
    p, n = randn(gen(1), (40, 9000), torch.float32), 30
    w = randn(gen(2), (9000, n), torch.float32)
    want, y = tg.linear(p, w), torch.empty(40, n, device="cuda")
    tg.lib.check(tg.lib.tg_linear(40, 9000, n, 0, p.data_ptr(), 9000, w.data_ptr(), n, 0, None, 0,
                                  None, 0, y.data_ptr(), n, None, 0, None, 0, tg.stream_handle()))
    assert torch.equal(y, want)
    dy = randn(gen(3), (40, n), torch.float32)
    dx, dw, db = tg.linear_backward(dy, p, w, bias=True)
    got = [torch.empty_like(v) for v in (dx, dw, db)]
    tg.lib.check(tg.lib.tg_linear_backward(
        40, 9000, n, 0, dy.data_ptr(), n, p.data_ptr(), 9000, w.data_ptr(), n, 0, None, 0, 0,
        got[0].data_ptr(), 9000, got[1].data_ptr(), got[2].data_ptr(), None, 0,
        tg.stream_handle()))
    assert all(torch.equal(a, b) for a, b in zip(got, (dx, dw, db)))
    r, value = tg.log_probs(p, torch.zeros(40, dtype=I32, device="cuda")), torch.empty(40,
                                                                                     device="cuda")
    z = randn(gen(4), (3, 70_000), torch.float32)
    labels = torch.tensor([5, 69_999, 0], dtype=I32, device="cuda")
    r, value = tg.log_probs(z, labels), torch.empty(3, device="cuda")
    tg.lib.check(tg.lib.tg_log_probs(3, 70_000, 0, z.data_ptr(), 70_000, labels.data_ptr(), 1.0, 0,
                                     value.data_ptr(), None, None, None, None, None, 0,
                                     tg.stream_handle()))
    assert torch.equal(value, r.value)


def test_written_inside_only(gpu):
    """Nothing behind the workspaces and the outputs."""
    import tinygnn_amd as tg

    def guarded(n):
        t = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        return t, lambda: bool((t[n:] == 0x5A).all())

    for rows, classes, k, top in ((3, 70_001, 5, 64), (2, 300_007, 200, 3), (700, 20_000, 9, 20)):
        for kind, dt in ((0, torch.float32), (1, torch.bfloat16)):
            z = randn(gen(classes), (rows, classes), dt)
            size = tg.lib.tg_log_probs_workspace_size(rows, classes, top, kind)
            ws, ok = guarded(size)
            tv, tv_ok = guarded(rows * top * 4)
            ti, ti_ok = guarded(rows * top * 4)
            tg.lib.check(tg.lib.tg_log_probs(
                rows, classes, kind, z.data_ptr(), classes, None, 1.0, top, None, None,
                tv.data_ptr(), ti.data_ptr(), None, ws.data_ptr(), size, tg.stream_handle()))
            assert ok() and tv_ok() and ti_ok()
            size = tg.lib.tg_distill_workspace_size(rows, classes, k, kind)
            ws, ok = guarded(size)
            d, d_ok = guarded(rows * classes * dt.itemsize)
            t = randn(gen(1), (rows, k), dt)
            ids = torch.randint(0, classes, (rows, k), device="cuda").to(I32)
            loss = torch.ones(rows, device="cuda")
            tg.lib.check(tg.lib.tg_distill(
                rows, classes, k, kind, z.data_ptr(), classes, kind, t.data_ptr(), ids.data_ptr(),
                1.0, loss.data_ptr(), torch.ones_like(loss).data_ptr(), d.data_ptr(), classes,
                ws.data_ptr(), size, tg.stream_handle()))
            assert ok() and d_ok()
    for m, k, n in ((40, 9000, 30), (3000, 260, 70), (700, 64, 640), (5000, 1024, 1280)):
        for kind, dt in ((0, torch.float32), (1, torch.bfloat16)):
            x, w, dy = (randn(gen(5), s, dt) for s in ((m, k), (k, n), (m, n)))
            size = tg.lib.tg_linear_workspace_size(m, k, n, kind)
            ws, ok = guarded(size)
            y, y_ok = guarded(m * n * dt.itemsize)
            tg.lib.check(tg.lib.tg_linear(m, k, n, kind, x.data_ptr(), k, w.data_ptr(), n, 0, None,
                                          4, None, 0, y.data_ptr(), n, None, 0, ws.data_ptr(),
                                          size, tg.stream_handle()))
            assert ok() and y_ok()
            size = tg.lib.tg_linear_backward_workspace_size(m, k, n, kind)
            ws, ok = guarded(size)
            dx, dx_ok = guarded(m * k * dt.itemsize)
            dw, dw_ok = guarded(k * n * dt.itemsize)
            db, db_ok = guarded(n * dt.itemsize)
            tg.lib.check(tg.lib.tg_linear_backward(
                m, k, n, kind, dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), n, 0,
                dy.data_ptr(), n, 4, dx.data_ptr(), k, dw.data_ptr(), db.data_ptr(), ws.data_ptr(),
                size, tg.stream_handle()))
            assert ok() and dx_ok() and dw_ok() and db_ok()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lead", [1, 2, 3, 5])
def test_any_alignment(gpu, dtype, lead):
    """Every operand and result `lead` elements into its memory: the bits of whole ones."""
    import tinygnn_amd as tg
    dt = DTYPES[dtype]

    def moved(t):
        wide = torch.full((t.numel() + lead + 8,), float("nan") if t.is_floating_point() else -7,
                          dtype=t.dtype, device="cuda")
        wide[lead:lead + t.numel()] = t.flatten()
        return wide[lead:lead + t.numel()].view(t.shape)

    def place(*shape):
        return moved(torch.zeros(shape, dtype=dt, device="cuda"))

    for m, k, n in ((3, 700, 1100), (33, 100, 41), (600, 520, 264)):
        g = gen(m + lead)
        for transpose in (False, True):
            x, w = randn(g, (m, k), dt), randn(g, (n, k) if transpose else (k, n), dt, k ** -0.5)
            b, r, dy = randn(g, n, dt), randn(g, (m, n), dt), randn(g, (m, n), dt)
            y = tg.linear(moved(x), moved(w), bias=moved(b), epilogue=tg.EPI_SILU,
                          residual=moved(r), transpose=transpose, out=place(m, n))
            want, tol, _, _ = hc.linear(x, w, b, "silu", r, transpose)
            within(y, want, hc.rounded(want, tol, dt), "y")
            got = tg.linear_backward(moved(dy), moved(x), moved(w), pre=moved(r),
                                     epilogue=tg.EPI_SILU, bias=True, transpose=transpose)
            ref = hc.linear_backward(dy, x, w, r, "silu", transpose, dt)
            for t, key in zip(got, ("dx", "dw", "db")):
                within(t, ref[key][0], hc.rounded(*ref[key], dt), key)
    for rows, classes in ((70, 41), (50, 300), (5, 20_003)):
        g = gen(classes + lead)
        z, dv = randn(g, (rows, classes), dt), randn(g, rows, torch.float32)
        labels = torch.randint(0, classes, (rows,), generator=g, device="cuda").to(I32)
        t, ids = randn(g, (rows, 5), dt), torch.randint(0, classes, (rows, 5), generator=g,
                                                        device="cuda").to(I32)
        a, c = (tg.log_probs(u, v, top=7, entropy=True) for u, v in
                ((z, labels), (moved(z), moved(labels))))
        for name in ("value", "entropy", "top_values", "top_ids"):
            assert torch.equal(getattr(a, name), getattr(c, name)), name
        assert torch.equal(tg.log_probs_backward(dv, z, labels, a),
                           tg.log_probs_backward(moved(dv), moved(z), moved(labels), c,
                                                 out=place(rows, classes)))
        for u, v in zip(tg.distill(z, t, ids, dloss=dv),
                        tg.distill(moved(z), moved(t), moved(ids), dloss=moved(dv),
                                   out=place(rows, classes))):
            assert torch.equal(u, v)


def test_far_rows(gpu):
    """Rows whose first element lies past 2^31 elements."""
    import tinygnn_amd as tg
    rows, classes = 33_000, 70_000     # 2.3e9 elements, 4.6 GB
    z = torch.zeros(rows, classes, dtype=torch.bfloat16, device="cuda")
    some = [0, 20_000, 30_700, 32_999]
    g = gen(7)
    part = randn(g, (len(some), classes), torch.bfloat16, 2.0)
    z[some] = part
    labels = torch.full((rows,), -1, dtype=I32, device="cuda")
    labels[some] = torch.tensor([3, 69_999, 40_000, 12], dtype=I32, device="cuda")
    few = labels[some].contiguous()
    ids = torch.randint(0, classes, (rows, 5), generator=g, device="cuda").to(I32)
    t, dv = randn(g, (rows, 5), torch.float32), torch.ones(rows, device="cuda")
    row = hc.Row(part, 1.0)
    r = tg.log_probs(z, labels, top=3, entropy=True)
    want, tol = hc.value(row, few)
    within(r.value[some], want, tol, "value")
    assert torch.equal(r.top_ids[some], hc.top(part, 3).to(I32))
    d = tg.log_probs_backward(dv, z, labels, r, out=z)
    ref, tol = hc.backward(row, few, dv[some], None, 1.0)
    within(d[some], ref, hc.rounded(ref, tol, torch.bfloat16), "dlogits")
    z[some] = part
    loss, d = tg.distill(z, t, ids, dloss=dv, out=z)
    want, tol, ref, dtol = hc.distill(row, t[some], ids[some], 1.0, dv[some])
    within(loss[some], want, tol, "loss")
    within(d[some], ref, hc.rounded(ref, dtol, torch.bfloat16), "distilled dlogits")


def test_far_layers(gpu):
    import tinygnn_amd as tg
    m, k, n = 300_000, 8192, 16        # x: 2.5e9 elements, 4.9 GB
    g = gen(8)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    some = [0, 150_000, 262_200, 299_999]
    part = randn(g, (len(some), k), torch.bfloat16)
    x[some] = part
    w, dy = randn(g, (n, k), torch.bfloat16, k ** -0.5), torch.zeros(m, n, dtype=torch.bfloat16,
                                                                     device="cuda")
    dy[some] = randn(g, (len(some), n), torch.bfloat16)
    y = tg.linear(x, w, transpose=True)
    want, tol, _, _ = hc.linear(part, w, None, "none", None, True)
    within(y[some], want, hc.rounded(want, tol, torch.bfloat16), "y")
    dx, dw, _ = tg.linear_backward(dy, x, w, transpose=True)
    ref = hc.linear_backward(dy[some], part, w, None, "none", True, torch.bfloat16)
    within(dx[some], ref["dx"][0], hc.rounded(*ref["dx"], torch.bfloat16), "dx")
    within(dw, ref["dw"][0], hc.rounded(*ref["dw"], torch.bfloat16), "dw")
