"""The expert-layer operators together, as a layer runs them: norm, router,
products in expert order, join, and back; on another stream; captured into a
graph and replayed; on two streams at once."""
import pytest
import torch

from expert_cases import gen, randn, within

pytestmark = pytest.mark.gpu

T, D, H, E, K = 700, 96, 160, 12, 3


def inputs(dtype, seed=3):
    g = gen(seed)
    p = dict(x=randn(g, (T, D), dtype), gamma=1 + randn(g, D, dtype, 0.1),
             beta=randn(g, D, dtype, 0.1), router=randn(g, (D, E), torch.float32, D ** -0.5),
             w1=randn(g, (E, D, H), dtype, D ** -0.5), b1=randn(g, (E, H), dtype, 0.1),
             w2=randn(g, (E, H, D), dtype, H ** -0.5), dout=randn(g, (T, D), dtype))
    p["x"][5] = 0
    return p


def forward_backward(tg, p, stream=None):
    """A pre-norm expert layer and its gradients; rows 7, 14, ... are padding
    (no expert)."""
    s = dict(stream=stream)
    xn, mean, rstd = tg.layer_norm(p["x"], p["gamma"], p["beta"], with_stats=True, **s)
    logits = tg.matmul(xn.float(), p["router"], **s)
    logits[7::7] = -float("inf")
    weights, experts, plan = tg.route(logits, K, renormalize=True, **s)
    h = torch.zeros(T * K, H, dtype=p["x"].dtype, device="cuda")
    tg.grouped_matmul(xn, p["w1"], plan.offsets, rows=plan.rows, bias=p["b1"],
                      epilogue=tg.EPI_RELU, out=h, **s)
    z = torch.zeros(T * K, D, dtype=p["x"].dtype, device="cuda")
    tg.grouped_matmul(h, p["w2"], plan.offsets, out=z, **s)
    out = tg.route_combine(z, plan.position, weights, **s)
    dz, dweights = tg.route_combine_backward(p["dout"], z, plan.position, weights,
                                             out=torch.zeros_like(z), **s)
    dh = torch.zeros_like(h)
    tg.grouped_matmul(dz, p["w2"], plan.offsets, transpose=True, out=dh, **s)
    dw2, _ = tg.grouped_matmul_wgrad(h, dz, plan.offsets, **s)
    dh = torch.where(h > 0, dh, torch.zeros_like(dh))
    dg = torch.zeros_like(z)
    tg.grouped_matmul(dh, p["w1"], plan.offsets, transpose=True, out=dg, **s)
    dw1, db1 = tg.grouped_matmul_wgrad(xn, dh, plan.offsets, rows=plan.rows, bias=True, **s)
    dlogits = tg.route_backward(dweights, logits, weights, experts, renormalize=True, **s)
    drouter = xn.float().t() @ dlogits
    dxn = tg.route_combine(dg, plan.position, **s) + (dlogits @ p["router"].t()).to(dg.dtype)
    dx, dgamma, dbeta = tg.layer_norm_backward(dxn, p["x"], mean, rstd, p["gamma"], **s)
    return dict(out=out, dx=dx, dgamma=dgamma, dbeta=dbeta, drouter=drouter, dw1=dw1, db1=db1,
                dw2=dw2, experts=experts, on=(h > 0)[plan.position.clamp_min(0).long()])


def reference(p, experts, on):
    """The same in 64 bits by torch's differentiation, the choices given: the
    experts, and the side of ReLU's corner (a value within a rounding of 0 may
    fall on either, and takes its row's whole term of a gradient with it)."""
    q = {k: v.double().requires_grad_(k != "dout") for k, v in p.items()}
    x = q["x"]
    d = x - x.mean(1, keepdim=True)
    xn = d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt() * q["gamma"] + q["beta"]
    live = experts[:, :1] >= 0
    logits = xn @ q["router"]
    chosen = torch.gather(logits, 1, experts.clamp_min(0).long())
    w = torch.where(live, torch.softmax(chosen, 1), 0.0)
    out = torch.zeros_like(x)
    for j in range(K):
        e = experts[:, j].clamp_min(0).long()
        h = (torch.bmm(xn[:, None], q["w1"][e])[:, 0] + q["b1"][e]) * on[:, j]
        out = out + w[:, j, None] * torch.bmm(h[:, None], q["w2"][e])[:, 0]
    names = ["x", "gamma", "beta", "router", "w1", "b1", "w2"]
    grads = torch.autograd.grad(out, [q[n] for n in names], p["dout"].double())
    return dict(out=out.detach(), **{"d" + n: g for n, g in zip(names, grads)})


@pytest.mark.parametrize("dtype,share", [(torch.float32, 2e-5), (torch.bfloat16, 6e-2)])
def test_layer(gpu, dtype, share):
    """share: of the largest gradient's size.  float32: sums of at most 2,100
    terms with some 400 u each way through seven operators, 7 * 400 * 2^-24 <
    2e-4 in the worst case, a tenth of it for sums of random signs; bf16: seven
    roundings of 2^-8 one after another, twice over for the pass back."""
    import tinygnn_amd as tg
    p = inputs(dtype)
    got = forward_backward(tg, p)
    want = reference(p, got["experts"], got["on"])
    assert bool((got["experts"][7::7] == -1).all()) and not got["out"][7::7].any()
    for name, v in want.items():
        within(got[name], v, share * v.abs().max(), name)


def test_layer_gradients_by_differences(gpu):
    """Each gradient g along its own direction against central differences of
    the plain forward pass in 64 bits.  Steps of 1e-6: the row of equal values
    has rstd 316, (316e-6)^2 < 1e-6 of the slope is left, and roundings of 2^-53
    of a sum of size 1e3 over 2e-6 less.  An error of `share` of the largest
    value in each of N places changes g's length by share * largest * sqrt(N)
    at most."""
    import tinygnn_amd as tg
    p, step, share = inputs(torch.float32), 1e-6, 2e-5
    got = forward_backward(tg, p)
    base = {k: v.double() for k, v in p.items()}
    for name in ("x", "gamma", "beta", "router", "w1", "b1", "w2"):
        g = got["d" + name].double()

        def loss(s):
            moved = {k: v.clone() for k, v in base.items()}
            moved[name] += s / g.norm() * g
            return (reference(moved, got["experts"], got["on"])["out"] * base["dout"]).sum()

        want = ((loss(step) - loss(-step)) / (2 * step)).item()
        tol = share * g.abs().max().item() * g.numel() ** 0.5 + 1e-6 * (1 + abs(want))
        assert abs(g.norm().item() - want) <= tol, (name, g.norm().item(), want, tol)


def test_layer_on_another_stream(gpu):
    """Inputs are finished; results of a stream that is not the current one are
    read at once."""
    import tinygnn_amd as tg
    p = inputs(torch.float32)
    want = forward_backward(tg, p)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            torch.mm(big, big)
    y, mean, rstd = tg.layer_norm(p["x"], p["gamma"], p["beta"], with_stats=True, stream=side)
    w0, m0, r0 = tg.layer_norm(p["x"], p["gamma"], p["beta"], with_stats=True)
    assert torch.equal(y, w0) and torch.equal(mean, m0) and torch.equal(rstd, r0)
    torch.cuda.synchronize()
    got = forward_backward(tg, p, stream=side)
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_layer_on_two_streams(gpu):
    """Two layers at once, each on its own stream: no shared workspace."""
    import tinygnn_amd as tg
    ps = [inputs(torch.bfloat16, seed) for seed in (3, 4)]
    want = [forward_backward(tg, p) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = forward_backward(tg, ps[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for name in w:
            assert torch.equal(g[name], w[name]), name


@pytest.mark.parametrize("tokens", [20, 3000])
def test_captured(gpu, tokens):
    """Captured, with torch memory as workspaces, and replayed on new inputs,
    eager calls of the same operators in between."""
    import tinygnn_amd as tg
    e, k, d, n = 20, 2, 64, 72

    def run(x, logits, w, dy):
        xn, mean, rstd = tg.layer_norm(x, with_stats=True)
        weights, experts, plan = tg.route(logits, k)
        y = tg.grouped_matmul(xn, w, plan.offsets, rows=plan.rows)
        out = tg.route_combine(y, plan.position, weights)
        dw, db = tg.grouped_matmul_wgrad(xn, dy, plan.offsets, rows=plan.rows, bias=True)
        dx, dgamma, dbeta = tg.layer_norm_backward(xn, x, mean, rstd)
        dl = tg.route_backward(weights, logits, weights, experts)
        types = tg.route_plan(experts, e)
        y8 = tg.matmul_fp8(tg.quantize(xn), tg.quantize_weight(w), offsets=plan.offsets,
                           rows=plan.rows)
        return [out, dw, db, dx, dgamma, dbeta, dl, types.position, y8, experts]

    def fresh(seed):
        g = gen(seed)
        return [randn(g, (tokens, d), torch.float32), randn(g, (tokens, e), torch.float32),
                randn(g, (e, d, n), torch.float32), randn(g, (tokens * k, n), torch.float32)]

    static = fresh(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(*static)
    for seed in (1, 2, 3):
        new = fresh(seed)
        want = run(*new)
        for s, v in zip(static, new):
            s.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), i


def test_capture_without_workspace_is_refused(gpu):
    """The C entries' own temporaries would outlive the call in the graph."""
    import tinygnn_amd as tg
    torch_ = gpu
    n, groups = 100_000, 8
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    out = [torch.empty(n + 1, dtype=torch.int32, device="cuda") for _ in range(3)]
    side = torch_.cuda.Stream()
    torch_.cuda.synchronize()
    graph = torch_.cuda.CUDAGraph()
    with torch_.cuda.stream(side):
        graph.capture_begin(capture_error_mode="relaxed")
        rc = tg.lib.tg_route_plan(n, groups, 1, ids.data_ptr(), out[0].data_ptr(),
                                  out[1].data_ptr(), out[2].data_ptr(), None, 0,
                                  int(side.cuda_stream))
        graph.capture_end()
    assert rc == 1 and b"being captured" in tg.lib.tg_last_error()


def test_typed_nodes(gpu):
    """A transform for each node type: the plan of the types, gathered rows, and
    back to the nodes' own order."""
    import tinygnn_amd as tg
    g, n, types = gen(5), 5000, 6
    x, w = randn(g, (n, 41), torch.float32), randn(g, (types, 41, 16), torch.float32)
    kind = torch.randint(0, types, (n,), generator=g, device="cuda", dtype=torch.int32)
    plan = tg.route_plan(kind, types)
    y = tg.grouped_matmul(x, w, plan.offsets, rows=plan.rows)
    out = tg.route_combine(y, plan.position.view(-1, 1))
    want = torch.bmm(x.double()[:, None], w.double()[kind.long()])[:, 0]
    size = torch.bmm(x.double().abs()[:, None], w.double().abs()[kind.long()])[:, 0]
    within(out, want, 43 * 2.0 ** -24 * size + 2.0 ** -24 * want.abs(), "out")
