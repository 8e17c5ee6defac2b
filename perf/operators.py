"""The dense operators of expert layers, as measurable cases.

A layer that sends each node (or token) to one or a few of many weight
matrices -- by a learned router, or by the node's type in a graph of several
types -- runs these, with the norm before it:

* ``norm``    -- ``tg.layer_norm`` and, in training, ``tg.layer_norm_backward``;
* ``route``   -- ``tg.route``: softmax, the k largest, and the order of the rows
  by expert; in training ``tg.route_backward``;
* ``combine`` -- ``tg.route_combine``: the weighted sum of each row's k results;
  in training ``tg.route_combine_backward``;
* ``grouped`` -- ``tg.grouped_matmul``: each group of rows times its own matrix;
  in training the gradients of x (the same product, transposed) and of the
  weights and biases (``tg.grouped_matmul_wgrad``);
* ``fp8``     -- ``tg.quantize`` and ``tg.matmul_fp8``: a served product in e4m3
  with a scale for each block of 128, one matrix or one for each group.

Every case makes its inputs on the GPU from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
E4M3_MAX = 448.0
BLOCK = 128


def listed():
    return [
        # The norm of one node's 256 hidden features, as in a query for a
        # single node: nothing but latency.
        dict(name="norm_one_row", op="norm", rows=1, cols=256, dtype="f32", train=False),
        # A training step's norm over every node of the 232,965-node graph at
        # its hidden width.
        dict(name="norm_233k_256", op="norm", rows=232_965, cols=256, dtype="f32", train=True),
        # ... and over a batch of wide bf16 rows.
        dict(name="norm_bf16_wide", op="norm", rows=16_384, cols=4096, dtype="bf16", train=True),
        # Routing of a handful of rows while serving.
        dict(name="route_8", op="route", tokens=8, experts=64, k=2, dtype="f32", renorm=True,
             masked=0.0, train=False),
        # Routing of a training batch over many experts, 8 for each row, some
        # rows padding.
        dict(name="route_64k_of_128", op="route", tokens=65_536, experts=128, k=8, dtype="bf16",
             renorm=False, masked=0.05, train=True),
        # Joining the results of 4 experts for each row, with its gradients.
        dict(name="combine_16k_2048", op="combine", tokens=16_384, k=4, cols=2048, dtype="bf16",
             train=True),
        # One transform for each of 7 node types over the 232,965-node graph's
        # 602 features (row stride of no 16 bytes), bias and ReLU, a training
        # step in fp32.
        dict(name="typed_233k_602_256", op="grouped", rows=232_965, groups=7, k=602, n=256,
             dtype="f32", top=1, skew=1.0, bias=True, epilogue="relu", train=True),
        # The up projection of an expert layer in a training step: 16,384 rows,
        # 2 of 32 experts for each, gathered by the router's order.
        dict(name="experts_bf16_train", op="grouped", rows=32_768, groups=32, k=2048, n=4096,
             dtype="bf16", top=2, skew=0.5, bias=False, epilogue="none", train=True),
        # The same layer serving 32 rows, 4 of 64 experts for each: the time to
        # read the weights.
        dict(name="experts_bf16_serve", op="grouped", rows=128, groups=64, k=2048, n=2048,
             dtype="bf16", top=4, skew=0.0, bias=True, epilogue="relu", train=False),
        # A wide product of a served batch in e4m3.
        dict(name="fp8_8k", op="fp8", rows=8192, groups=0, k=4096, n=8192, dtype="bf16", top=1,
             skew=0.0, bias=False, epilogue="none"),
        # ... of a few rows,
        dict(name="fp8_5_rows", op="fp8", rows=5, groups=0, k=4096, n=4096, dtype="bf16", top=1,
             skew=0.0, bias=True, epilogue="none"),
        # ... and of a batch of 4,096 rows over 16 experts.
        dict(name="fp8_experts", op="fp8", rows=4096, groups=16, k=2048, n=4096, dtype="bf16",
             top=2, skew=0.5, bias=False, epilogue="none"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: an operator, and sizes log-uniform over its range."""
    op = rng.choice(["norm", "norm", "route", "route", "combine", "grouped", "grouped", "grouped",
                     "fp8", "fp8"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "norm":
        rows, cols = _log(rng, 1, 250_000), _log(rng, 16, 8192)
        rows = max(1, min(rows, 67_000_000 // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, train=rng.random() < 0.7)
    if op == "route":
        experts = _log(rng, 4, 256)
        return dict(op=op, tokens=_log(rng, 1, 65_536), experts=experts,
                    k=rng.randint(1, min(8, experts)), dtype=dtype, renorm=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.1, 0.5]), train=rng.random() < 0.6)
    if op == "combine":
        tokens, k = _log(rng, 1, 65_536), rng.randint(1, 8)
        cols = _log(rng, 16, 4096)
        cols = max(16, min(cols, 134_000_000 // (tokens * k)))
        return dict(op=op, tokens=tokens, k=k, cols=cols, dtype=dtype, train=rng.random() < 0.6)
    top = rng.choice([1, 1, 2, 4])
    rows = top * _log(rng, 1, 60_000)
    # whole 16-element rows mostly, as layers have them, and any width else
    step = rng.choice([1, 16, 16, 64])
    k, n = (max(step, _log(rng, 16, 4096) // step * step) for _ in range(2))
    epilogue = rng.choice(["none", "none", "relu", "elu"])
    if op == "grouped":
        groups = _log(rng, 2, 64)
        train = rng.random() < 0.6
        most = 2.5e11 if dtype != "f32" else 3e10
        while rows * k * n > most or rows * max(k, n) > 2.5e8:
            rows = max(top, rows // 2 // top * top)
        return dict(op=op, rows=rows, groups=groups, k=k, n=n, dtype=dtype, top=top,
                    skew=rng.choice([0.0, 0.5, 1.5]), bias=rng.random() < 0.5, epilogue=epilogue,
                    train=train)
    groups = rng.choice([0, 0, _log(rng, 2, 32)])
    top = top if groups else 1
    rows = rows // top * top or top
    while rows * k * n > 2.7e11 or rows * max(k, n) > 2e8:
        rows = max(top, rows // 2 // top * top)
    return dict(op=op, rows=rows, groups=groups, k=k, n=n, dtype=dtype, top=top,
                skew=rng.choice([0.0, 0.5, 1.5]), bias=rng.random() < 0.5, epilogue=epilogue)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(TYPES[dtype])


def _sizes(groups, rows, skew, seed):
    """Rows of each group: shares falling as a power of a random rank (the
    few popular experts, the common node types), the last ones often empty."""
    r = torch.Generator().manual_seed(seed)
    share = (torch.randperm(groups, generator=r) + 1).double() ** -skew
    share = share * (0.5 + torch.rand(groups, generator=r, dtype=torch.float64))
    who = torch.multinomial(share, rows, replacement=True, generator=r)
    return torch.bincount(who, minlength=groups)


def _groups(case, seed, g):
    """What the router's plan holds: offsets, the row of x behind each row in
    expert order, and the place of each (row, choice) in that order."""
    rows, groups, top = case["rows"], case["groups"], case["top"]
    sizes = _sizes(groups, rows, case["skew"], seed)
    offsets = torch.zeros(groups + 1, dtype=torch.int64)
    offsets[1:] = sizes.cumsum(0)
    slot = torch.randperm(rows, generator=g, device=DEV)   # slot (row * top + choice) of each row
    place = torch.empty_like(slot)
    place[slot] = torch.arange(rows, device=DEV)
    return dict(sizes=sizes.tolist(), offsets=offsets.to(DEV, torch.int32),
                index=(slot // top).to(torch.int32) if top > 1 else None,
                position=place.to(torch.int32).view(-1, top))


def _block_quantized(w):
    """w [.., n, k] as e4m3 values [.., n, whole blocks of k] and the scale of
    each 128 x 128 block, the form in which checkpoints hold them."""
    n, k = w.shape[-2:]
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    lead = w.shape[:-2]
    full = torch.zeros(*lead, nb * BLOCK, kb * BLOCK, device=DEV)
    full[..., :n, :k] = w
    blocks = full.view(*lead, nb, BLOCK, kb, BLOCK)
    scale = (blocks.abs().amax((-3, -1)) / E4M3_MAX).clamp_min(torch.finfo(torch.float32).tiny)
    q = (blocks / scale[..., :, None, :, None]).view_as(full)[..., :n, :]
    return q.contiguous().to(torch.float8_e4m3fn), scale.contiguous()


def prepare(case, seed):
    op, dtype = case["op"], case["dtype"]
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if op == "norm":
        shape = (case["rows"], case["cols"])
        # features with an offset and a spread of their own in each column
        s["x"] = (torch.randn(shape, generator=g, device=DEV)
                  * (0.5 + torch.rand(shape[1], generator=g, device=DEV))
                  + 0.3 * torch.randn(shape[1], generator=g, device=DEV)).to(TYPES[dtype])
        s["gamma"] = (1 + 0.2 * torch.randn(shape[1], generator=g, device=DEV)).to(TYPES[dtype])
        s["beta"] = _normal(g, shape[1], dtype, 0.2)
        if case["train"]:
            s["dy"] = _normal(g, shape, dtype)
    elif op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        logits = torch.randn((t, e), generator=g, device=DEV) * 1.5
        if case["masked"]:
            # padded rows may go nowhere, and some experts are full
            logits[torch.rand(t, generator=g, device=DEV) < case["masked"]] = -math.inf
            logits[torch.rand((t, e), generator=g, device=DEV) < 0.02] = -math.inf
        s["logits"] = logits.to(TYPES[dtype])
        if case["train"]:
            s["dw"] = torch.randn((t, k), generator=g, device=DEV)
    elif op == "combine":
        t, k, c = case["tokens"], case["k"], case["cols"]
        s["y"] = _normal(g, (t * k, c), dtype)
        w = torch.rand((t, k), generator=g, device=DEV) + 0.05
        s["w"] = w / w.sum(1, keepdim=True)
        s["position"] = torch.randperm(t * k, generator=g, device=DEV).to(torch.int32).view(t, k)
        if case["train"]:
            s["dout"] = _normal(g, (t, c), dtype)
    else:
        k, n, groups = case["k"], case["n"], case["groups"]
        many = (groups,) if groups else ()
        s["x"] = _normal(g, (case["rows"] // case["top"], k), dtype)
        w = torch.randn((*many, k, n), generator=g, device=DEV) / math.sqrt(k)
        s["bias"] = _normal(g, (*many, n), dtype, 0.1) if case["bias"] else None
        if groups:
            s.update(_groups(case, seed, g))
        if op == "fp8":
            s["wq"], s["ws"] = _block_quantized(w.transpose(-1, -2))
        else:
            s["w"] = w.to(TYPES[dtype])
            if case["train"]:
                s["dy"] = _normal(g, (case["rows"], n), dtype)
    return s


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _own_run(s):
    import tinygnn_amd as tg
    case = s["case"]
    op = case["op"]
    if op == "norm":
        if not case["train"]:
            return dict(y=tg.layer_norm(s["x"], s["gamma"], s["beta"], EPS))
        y, mean, rstd = tg.layer_norm(s["x"], s["gamma"], s["beta"], EPS, with_stats=True)
        dx, dgamma, dbeta = tg.layer_norm_backward(s["dy"], s["x"], mean, rstd, s["gamma"])
        return dict(y=y, dx=dx, dgamma=dgamma, dbeta=dbeta)
    if op == "route":
        w, experts, plan = tg.route(s["logits"], case["k"], renormalize=case["renorm"])
        out = dict(w=w, experts=experts, offsets=plan.offsets, rows=plan.rows,
                   position=plan.position)
        if case["train"]:
            out["dlogits"] = tg.route_backward(s["dw"], s["logits"], w, experts,
                                               renormalize=case["renorm"])
        return out
    if op == "combine":
        out = dict(out=tg.route_combine(s["y"], s["position"], s["w"]))
        if case["train"]:
            out["dy"], out["dw"] = tg.route_combine_backward(s["dout"], s["y"], s["position"],
                                                             s["w"])
        return out
    epilogue = dict(none=tg.EPI_NONE, relu=tg.EPI_RELU, elu=tg.EPI_ELU)[case["epilogue"]]
    if op == "fp8":
        xq = tg.quantize(s["x"])
        wq = tg.BlockWeight(s["wq"], s["ws"], case["k"])
        return dict(y=tg.matmul_fp8(xq, wq, offsets=s.get("offsets"), rows=s.get("index"),
                                    bias=s["bias"], epilogue=epilogue, dtype=s["x"].dtype))
    out = dict(y=tg.grouped_matmul(s["x"], s["w"], s["offsets"], rows=s["index"], bias=s["bias"],
                                   epilogue=epilogue))
    if case["train"]:
        dx = tg.grouped_matmul(s["dy"], s["w"], s["offsets"], transpose=True)
        out["dx"] = tg.route_combine(dx, s["position"])
        out["dw"], out["db"] = tg.grouped_matmul_wgrad(s["x"], s["dy"], s["offsets"],
                                                       rows=s["index"], bias=case["bias"])
    return out


# ---------------------------------------------------------------------------
# Their plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------
def _epilogue(v, bias, epilogue):
    if bias is not None:
        v = v + bias
    if epilogue == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    return torch.where(v < 0, torch.exp(v) - 1, v) if epilogue == "elu" else v


def _norm_plain(s):
    x, gamma = s["x"].float(), s["gamma"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d * r
    out = dict(y=(xh * gamma + s["beta"].float()).to(s["x"].dtype))
    if s["case"]["train"]:
        dy = s["dy"].float()
        t = dy * gamma
        dx = r * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
        out["dx"] = dx.to(s["x"].dtype)
        out["dgamma"] = (dy * xh).sum(0).to(s["gamma"].dtype)
        out["dbeta"] = dy.sum(0).to(s["gamma"].dtype)
    return out


def _route_plain(s):
    case, k = s["case"], s["case"]["k"]
    x = s["logits"].float()
    t, e = x.shape
    # the k largest, the lower index first among equals
    chosen = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    live = torch.gather(x, 1, chosen) > -math.inf
    top = x.max(1, keepdim=True)[0]
    p = torch.where(x > -math.inf, torch.exp(x - top), torch.zeros_like(x))
    total = p.sum(1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    w = torch.gather(p, 1, chosen)
    if case["renorm"]:
        part = w.sum(1, keepdim=True)
        w = torch.where(part > 0, w / part, torch.zeros_like(w))
    experts = torch.where(live, chosen, torch.full_like(chosen, -1)).to(torch.int32)
    # rows in expert order; what goes nowhere comes last
    ids = torch.where(live, chosen, torch.full_like(chosen, e)).reshape(-1)
    by, slot = torch.sort(ids, stable=True)
    offsets = torch.searchsorted(by, torch.arange(e + 1, device=DEV))
    none = torch.full_like(slot, -1)
    position = torch.empty_like(slot)
    position[slot] = torch.where(by < e, torch.arange(t * k, device=DEV), none)
    out = dict(w=w, experts=experts, offsets=offsets.to(torch.int32),
               rows=torch.where(by < e, slot // k, none).to(torch.int32),
               position=position.view(t, k).to(torch.int32))
    if case["train"]:
        dw = torch.where(live, s["dw"], torch.zeros_like(s["dw"]))
        inner = (dw * w).sum(1, keepdim=True)
        if case["renorm"]:
            dl = torch.zeros_like(x).scatter_(1, chosen, w * (dw - inner))
        else:
            dl = p * (torch.zeros_like(x).scatter_(1, chosen, dw) - inner)
        out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _combine_plain(s):
    y, w, at = s["y"].float(), s["w"], s["position"].long()
    mine = y[at]
    out = dict(out=(mine * w[:, :, None]).sum(1).to(s["y"].dtype))
    if s["case"]["train"]:
        dout = s["dout"].float()[:, None, :]
        dy = torch.empty_like(y)
        dy[at] = w[:, :, None] * dout
        out["dy"] = dy.to(s["y"].dtype)
        out["dw"] = (mine * dout).sum(2)
    return out


def _grouped_plain(s):
    case = s["case"]
    x, w = s["x"].float(), s["w"].float()
    kind = s["x"].dtype
    if s["index"] is not None:
        x = x[s["index"].long()]
    xs = x.split(s["sizes"])
    y = torch.cat([a @ b for a, b in zip(xs, w)])
    group = torch.repeat_interleave(torch.arange(case["groups"], device=DEV),
                                    torch.diff(s["offsets"].long()), output_size=case["rows"])
    bias = s["bias"].float()[group] if case["bias"] else None
    out = dict(y=_epilogue(y, bias, case["epilogue"]).to(kind))
    if case["train"]:
        dys = s["dy"].float().split(s["sizes"])
        dx = torch.cat([a @ b.t() for a, b in zip(dys, w)])
        # each row's gradient in the inputs' type, then their sum over its copies
        out["dx"] = dx.to(kind).float()[s["position"].long()].sum(1).to(kind)
        out["dw"] = torch.stack([a.t() @ b for a, b in zip(xs, dys)]).to(kind)
        out["db"] = torch.stack([b.sum(0) for b in dys]).to(kind) if case["bias"] else None
    return out


def _quantized_plain(x):
    """The values that x [rows, k] stands for in e4m3, a scale for each row
    and 128 columns."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    full = torch.zeros(rows, kb * BLOCK, device=DEV)
    full[:, :k] = x
    blocks = full.view(rows, kb, BLOCK)
    scale = (blocks.abs().amax(2, keepdim=True) / E4M3_MAX).clamp_min(
        torch.finfo(torch.float32).tiny)
    q = (blocks / scale).to(torch.float8_e4m3fn)
    return (q.float() * scale).view(rows, -1)


def _weights_plain(s):
    q, scale = s["wq"], s["ws"]
    n = q.shape[-2]
    wide = scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)
    return q.float() * wide


def _fp8_plain(s):
    case = s["case"]
    x, w = _quantized_plain(s["x"].float()), _weights_plain(s)
    bias = s["bias"].float() if case["bias"] else None
    if case["groups"]:
        if s["index"] is not None:
            x = x[s["index"].long()]
        y = torch.cat([a @ b.t() for a, b in zip(x.split(s["sizes"]), w)])
        if case["bias"]:
            group = torch.repeat_interleave(torch.arange(case["groups"], device=DEV),
                                            torch.diff(s["offsets"].long()),
                                            output_size=case["rows"])
            bias = bias[group]
    else:
        y = x @ w.t()
    return dict(y=_epilogue(y, bias, case["epilogue"]).to(s["x"].dtype))


def run(state):
    if own:
        return _own_run(state)
    return dict(norm=_norm_plain, route=_route_plain, combine=_combine_plain,
                grouped=_grouped_plain, fp8=_fp8_plain)[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# The work of a pass, and its outputs from the definitions in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op, z = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        r, c = case["rows"], case["cols"]
        if not case["train"]:
            return dict(bytes=z * (2 * r * c + 2 * c), flops=8 * r * c)
        # the training step reads x and dy and writes y and dx
        return dict(bytes=z * (4 * r * c + 5 * c) + 8 * r, flops=22 * r * c)
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        b, f = z * t * e + 4 * (4 * t * k + e + 1), (4 + k) * t * e
        if case["train"]:
            b, f = b + z * t * e + 4 * t * k, f + 4 * t * e
        return dict(bytes=b, flops=f)
    if op == "combine":
        t, k, c = case["tokens"], case["k"], case["cols"]
        b, f = z * (t * k * c + t * c) + 8 * t * k, 2 * t * k * c
        if case["train"]:
            b, f = b + z * (t * c + t * k * c) + 4 * t * k, f + 3 * t * k * c
        return dict(bytes=b, flops=f)
    rows, k, n, top = case["rows"], case["k"], case["n"], case["top"]
    many = max(1, min(case["groups"], rows))
    if op == "fp8":
        return dict(bytes=z * (rows // top * k + rows * n) + many * n * k, flops=2 * rows * k * n)
    b, f = z * (rows // top * k + many * k * n + rows * n), 2 * rows * k * n
    if case["train"]:
        # x, w and dy read; y, dx and dw written
        b = z * (2 * (rows // top) * k + 2 * many * k * n + 2 * rows * n)
        f *= 3
    return dict(bytes=b, flops=f)


def _e4m3(v):
    """v (64 bits, at most 448 in size) to the nearest e4m3 value, ties to
    even: steps of 2^-3 of the leading power of two, 2^-9 at least."""
    power = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    power = power + (v.abs() >= 2.0 ** (power + 1)).double() - (v.abs() < 2.0 ** power).double()
    step = 2.0 ** (power.clamp_min(-6.0) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, g = s["x"].double(), s["gamma"].double()
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        xh = (x - mean) / (var + EPS).sqrt()
        out = dict(y=xh * g + s["beta"].double())
        if case["train"]:
            dy = s["dy"].double()
            c = x.shape[1]
            # the projection of the scaled gradient off the ones and off xh
            t = dy * g
            off = (t.sum(1, keepdim=True) + xh * torch.einsum("rc,rc->r", t, xh)[:, None]) / c
            out.update(dx=(t - off) / (var + EPS).sqrt(),
                       dgamma=torch.einsum("rc,rc->c", dy, xh), dbeta=dy.sum(0))
        return out
    if op == "route":
        x, k = s["logits"].double(), case["k"]
        t, e = x.shape
        rank = x.clone()
        picks = []
        for _ in range(k):   # the largest left, the lowest index among equals
            best = rank.max(1, keepdim=True)[0]
            first = torch.where(rank == best, torch.arange(e, device=DEV), e).min(1)[0]
            picks.append(torch.where(best[:, 0] > -math.inf, first, -1))
            rank[torch.arange(t, device=DEV), first] = -math.inf
        chosen = torch.stack(picks, 1)
        live = chosen >= 0
        p = torch.nan_to_num(torch.exp(x - torch.logsumexp(x, 1, keepdim=True)), nan=0.0)
        w = torch.where(live, torch.gather(p, 1, chosen.clamp_min(0)), 0.0)
        scale = torch.ones_like(w[:, :1])
        if case["renorm"]:
            scale = w.sum(1, keepdim=True)
            scale = torch.where(scale > 0, scale, 1.0)
        w = w / scale
        slots = torch.arange(t * k, device=DEV)
        ids = torch.where(live, chosen, e).reshape(-1)
        order = torch.argsort(ids * (t * k) + slots)
        kept = int(live.sum())
        rows = torch.full_like(slots, -1)
        rows[:kept] = order[:kept] // k
        position = torch.full_like(slots, -1)
        position[order[:kept]] = slots[:kept]
        out = dict(w=w, experts=chosen.int(), rows=rows.int(), position=position.view(t, k).int(),
                   offsets=torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV),
                                      torch.bincount(ids, minlength=e + 1)[:e].cumsum(0)]).int())
        if case["train"]:
            dw = torch.where(live, s["dw"].double(), 0.0)
            hit = torch.zeros(t, e + 1, dtype=torch.float64, device=DEV)
            hit.scatter_(1, torch.where(live, chosen, e), dw)
            over = p
            if case["renorm"]:
                keep = torch.zeros(t, e + 1, dtype=torch.float64, device=DEV)
                keep.scatter_(1, torch.where(live, chosen, e), 1.0)
                over = p * keep[:, :e] / scale
            out["dlogits"] = over * (hit[:, :e] - (dw * w).sum(1, keepdim=True))
        return out
    if op == "combine":
        t, k, c = case["tokens"], case["k"], case["cols"]
        flat, w = s["position"].long().reshape(-1), s["w"].double()
        y = s["y"].double()
        out = dict(out=torch.zeros(t, c, dtype=torch.float64, device=DEV))
        for j in range(k):
            out["out"] += w[:, j, None] * y[s["position"][:, j].long()]
        if case["train"]:
            dout = s["dout"].double()
            token = torch.empty_like(flat)
            token[flat] = torch.arange(t * k, device=DEV)
            out["dy"] = dout[token // k] * w.reshape(-1)[token, None]
            dots = torch.empty(t * k, dtype=torch.float64, device=DEV)
            dots[token] = (dout[token // k] * y).sum(1)
            out["dw"] = dots.view(t, k)
        return out
    x, off = s["x"], s.get("offsets")
    if op == "fp8":
        pad = -case["k"] % BLOCK
        x = torch.nn.functional.pad(x.float(), (0, pad)).view(x.shape[0], -1, BLOCK)
        # scale and quotient are rounded to 32 bits by definition
        scale = torch.maximum(x.abs().max(2, keepdim=True)[0] / E4M3_MAX,
                              torch.full((1, 1, 1), 2.0 ** -126, device=DEV))
        x = (_e4m3((x / scale).double()) * scale.double()).flatten(1)
        at = torch.arange(case["n"], device=DEV) // BLOCK
        w = s["wq"].double().unflatten(-1, (-1, BLOCK)) * s["ws"].double()[..., at, :, None]
        w = w.flatten(-2).transpose(-1, -2)
    else:
        x, w = x.double(), s["w"].double()
    if not case["groups"]:
        off, w = torch.tensor([0, case["rows"]]), w[None]
    if s.get("index") is not None:
        x = x[s["index"].long()]
    off = off.tolist()
    y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=DEV)
    out = dict(y=y)
    if case.get("train"):
        dx = torch.empty(case["rows"], case["k"], dtype=torch.float64, device=DEV)
        out["dw"] = torch.empty_like(w)
        out["db"] = torch.empty(len(off) - 1, case["n"], dtype=torch.float64, device=DEV)
    for i, (lo, hi) in enumerate(zip(off, off[1:])):
        y[lo:hi] = x[lo:hi] @ w[i]
        if case["bias"]:
            y[lo:hi] += (s["bias"][i] if case["groups"] else s["bias"]).double()
        if case.get("train"):
            dy = s["dy"][lo:hi].double()
            dx[lo:hi] = dy @ w[i].t()
            out["dw"][i] = x[lo:hi].t() @ dy
            out["db"][i] = dy.sum(0)
    if case["epilogue"] == "relu":
        y.clamp_min_(0.0)
    elif case["epilogue"] == "elu":
        out["y"] = torch.where(y < 0, torch.expm1(y), y)
    if case.get("train"):
        out["dx"] = torch.zeros(case["rows"] // case["top"], case["k"], dtype=torch.float64,
                                device=DEV)
        for j in range(case["top"]):
            out["dx"] += dx[s["position"][:, j].long()]
        if not case["bias"]:
            out["db"] = None
    return out
