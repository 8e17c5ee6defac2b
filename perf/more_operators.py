"""The operators of a classifier's head and of what it learns from, as measurable cases.

A graph's network is often served, and distilled, as plain dense layers over
the nodes' features; those layers and their losses run these:

* ``linear``  -- ``tg.linear``: a dense product with bias, activation and
  residual in its epilogue; in training ``tg.linear_backward``;
* ``logp``    -- ``tg.log_probs``: the log probability of each row's given
  class, the entropy, and the likeliest classes; in training
  ``tg.log_probs_backward``;
* ``distill`` -- ``tg.distill``: the divergence from a teacher's top logits; in
  training with its gradient.

Every case makes its inputs on the GPU from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
GELU_CUBE = 0.044715


def listed():
    return [
        # One node's hidden features through one wide layer while serving: the
        # time to read the weights, kept [n, k] as checkpoints hold them.
        dict(name="linear_one_row", op="linear", rows=1, k=4096, n=4096, dtype="bf16", bias=True,
             epilogue="silu", residual=False, transpose=True, train=False),
        # A few queries at once, onto the residual stream, weights [k, n].
        dict(name="linear_12_rows", op="linear", rows=12, k=8192, n=2048, dtype="f16", bias=False,
             epilogue="none", residual=True, transpose=False, train=False),
        # A training step of a residual hidden layer over all nodes of the
        # 232,965-node graph, in fp32.
        dict(name="linear_233k_256", op="linear", rows=232_965, k=256, n=256, dtype="f32",
             bias=True, epilogue="elu", residual=True, transpose=False, train=True),
        # A training step of a wide layer's up projection.
        dict(name="linear_bf16_train", op="linear", rows=16_384, k=2048, n=8192, dtype="bf16",
             bias=True, epilogue="gelu", residual=False, transpose=False, train=True),
        # A served batch's down projection onto the residual stream; rows of no
        # whole tile.
        dict(name="linear_bf16_down", op="linear", rows=4000, k=8192, n=2048, dtype="bf16",
             bias=True, epilogue="none", residual=True, transpose=True, train=False),
        # What a server answers for one row: its class's log probability and 20
        # alternatives of many.
        dict(name="logp_one_row", op="logp", rows=1, classes=131_072, dtype="f32", top=20,
             entropy=True, temperature=1.0, train=False),
        # ... and for a batch of 64.
        dict(name="logp_64_top", op="logp", rows=64, classes=100_003, dtype="f16", top=20,
             entropy=False, temperature=0.7, train=False),
        # The cross entropy of 41 classes over the 232,965 nodes, with an
        # entropy term, and its gradient.
        dict(name="logp_233k_41", op="logp", rows=232_965, classes=41, dtype="f32", top=0,
             entropy=True, temperature=1.0, train=True),
        # ... of 32,000 classes over a batch of rows.
        dict(name="logp_8k_32k", op="logp", rows=8192, classes=32_000, dtype="bf16", top=0,
             entropy=False, temperature=1.0, train=True),
        # Distillation of a graph's network into dense layers: 8 of 41 classes
        # kept for each of the 232,965 nodes.
        dict(name="distill_233k_41", op="distill", rows=232_965, classes=41, k=8, dtype="f32",
             temperature=2.0, train=True),
        # ... of 65,536 classes, 32 kept.
        dict(name="distill_4k_64k", op="distill", rows=4096, classes=65_536, k=32, dtype="bf16",
             temperature=1.0, train=True),
        # The loss alone, over a small held-out set.
        dict(name="distill_300_eval", op="distill", rows=300, classes=50_001, k=16, dtype="f32",
             temperature=1.0, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: an operator, and sizes log-uniform over its range."""
    op = rng.choice(["linear", "linear", "linear", "logp", "logp", "logp", "distill", "distill"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "linear":
        rows = _log(rng, 1, 250_000)
        # whole 16-element rows mostly, as layers have them, and any width else
        step = rng.choice([1, 16, 16, 64])
        k, n = (max(step, _log(rng, 16, 8192) // step * step) for _ in range(2))
        most = 2.7e11 if dtype != "f32" else 1.5e10
        while rows * k * n > most or rows * max(k, n) > 1.3e8:
            rows = max(1, rows // 2)
        train = rng.random() < 0.5
        # ReLU's slope jumps at 0: the last bits of a 32-bit sum decide there, and
        # a row's whole gradient goes with it.  Below a 16-bit rounding, above fp32's.
        some = ["none", "elu", "gelu", "silu"] + ["relu"] * (not train or dtype != "f32")
        return dict(op=op, rows=rows, k=k, n=n, dtype=dtype, bias=rng.random() < 0.6,
                    epilogue=rng.choice(some), residual=rng.random() < 0.5,
                    transpose=rng.random() < 0.5, train=train)
    classes = _log(rng, 2, 131_072)
    rows = max(1, min(_log(rng, 1, 250_000), 260_000_000 // classes))
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    train = rng.random() < 0.5
    if op == "distill":
        return dict(op=op, rows=rows, classes=classes, k=min(classes, _log(rng, 1, 64)),
                    dtype=dtype, temperature=temperature, train=train)
    return dict(op=op, rows=rows, classes=classes, dtype=dtype,
                top=min(classes, rng.choice([0, 0, 1, 5, 20, 32])), entropy=rng.random() < 0.5,
                temperature=temperature, train=train)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(TYPES[dtype])


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device=DEV)


def _whole(g, high, *shape):
    return torch.randint(high, shape, generator=g, device=DEV)


def prepare(case, seed):
    op, dtype, rows = case["op"], case["dtype"], case["rows"]
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if op == "linear":
        k, n = case["k"], case["n"]
        s["x"] = _normal(g, (rows, k), dtype)
        s["w"] = _normal(g, (n, k) if case["transpose"] else (k, n), dtype, k ** -0.5)
        s["bias"] = _normal(g, n, dtype, 0.1) if case["bias"] else None
        s["residual"] = _normal(g, (rows, n), dtype) if case["residual"] else None
        if case["train"]:
            s["dy"] = _normal(g, (rows, n), dtype)
        return s
    # logits: some classes commoner than others, rows of more and less certainty
    c = case["classes"]
    logits = torch.randn((rows, c), generator=g, device=DEV)
    logits *= 0.5 + 2.0 * _uniform(g, rows, 1)
    logits += torch.randn(c, generator=g, device=DEV)
    # each row's own class, mostly near the front, never a masked one
    labels = _whole(g, c, rows)
    logits[torch.arange(rows, device=DEV), labels] += 3.0
    if c >= 64:
        mask = _uniform(g, rows, c) < 0.02
        mask[torch.arange(rows, device=DEV), labels] = False
        logits[mask] = -math.inf
        del mask
    s["logits"] = logits.to(TYPES[dtype])
    scale = 1024.0 if dtype == "f16" else 1.0     # as 16-bit losses are scaled
    if op == "logp":
        labels = torch.where(_uniform(g, rows) < 0.05, -1, labels)   # rows without a class
        s["labels"] = labels.to(torch.int32)
        if case["train"]:
            s["dvalue"] = -scale * (0.5 + _uniform(g, rows))
            s["dentropy"] = 0.1 * scale * _uniform(g, rows) if case["entropy"] else None
        return s
    teacher = logits + 0.7 * torch.randn((rows, c), generator=g, device=DEV)
    top, ids = torch.topk(teacher, case["k"], 1)
    # the teacher's file keeps its values in 16 bits where the student's are;
    # a few places are empty
    none = _uniform(g, rows, case["k"]) < 0.02
    none[:, 0] = False
    s["teacher"] = top.to(TYPES[dtype])
    s["ids"] = torch.where(none, -1, ids).to(torch.int32)
    if case["train"]:
        s["dloss"] = scale * (_uniform(g, rows) < 0.95).float() * case["temperature"] ** 2
    return s


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _own_run(s):
    import tinygnn_amd as tg
    case = s["case"]
    if case["op"] == "linear":
        epilogue = dict(none=tg.EPI_NONE, relu=tg.EPI_RELU, elu=tg.EPI_ELU, gelu=tg.EPI_GELU,
                        silu=tg.EPI_SILU)[case["epilogue"]]
        plain = epilogue == tg.EPI_NONE
        kept = case["train"] and not plain
        y = tg.linear(s["x"], s["w"], bias=s["bias"], epilogue=epilogue, residual=s["residual"],
                      transpose=case["transpose"], with_pre=kept)
        y, pre = y if kept else (y, None)
        out = dict(y=y)
        if case["train"]:
            out["dx"], out["dw"], db = tg.linear_backward(
                s["dy"], s["x"], s["w"], pre=pre, epilogue=epilogue, bias=case["bias"],
                transpose=case["transpose"])
            if case["bias"]:
                out["db"] = db
        return out
    if case["op"] == "logp":
        r = tg.log_probs(s["logits"], s["labels"], top=case["top"], entropy=case["entropy"],
                         temperature=case["temperature"])
        out = dict(value=r.value)
        if case["entropy"]:
            out["entropy"] = r.entropy
        if case["top"]:
            out.update(top_values=r.top_values, top_ids=r.top_ids)
        if case["train"]:
            out["dlogits"] = tg.log_probs_backward(s["dvalue"], s["logits"], s["labels"], r,
                                                   dentropy=s["dentropy"],
                                                   temperature=case["temperature"])
        return out
    r = tg.distill(s["logits"], s["teacher"], s["ids"], temperature=case["temperature"],
                   dloss=s.get("dloss"))
    return dict(loss=r[0], dlogits=r[1]) if case["train"] else dict(loss=r)


# ---------------------------------------------------------------------------
# Their plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------
def _sigmoid(v):
    e = torch.exp(-v.abs())
    return torch.where(v < 0, e, torch.ones_like(e)) / (1 + e)


def _inner(v):
    return math.sqrt(8 / math.pi) * (v + GELU_CUBE * v * v * v)


def _act_plain(v, epilogue):
    if epilogue == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if epilogue == "elu":
        return torch.where(v < 0, torch.exp(v) - 1, v)
    if epilogue == "gelu":      # 0.5 v (1 + tanh(u)) = v sigmoid(2 u)
        return v * _sigmoid(_inner(v))
    return v * _sigmoid(v) if epilogue == "silu" else v


def _slope_plain(v, epilogue):
    if epilogue == "relu":
        return (v > 0).to(v.dtype)
    if epilogue == "elu":
        return torch.where(v < 0, torch.exp(v), torch.ones_like(v))
    if epilogue == "gelu":
        p = _sigmoid(_inner(v))
        return p + v * p * (1 - p) * math.sqrt(8 / math.pi) * (1 + 3 * GELU_CUBE * v * v)
    p = _sigmoid(v)
    return p + v * p * (1 - p)


def _linear_plain(s):
    case = s["case"]
    kind = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    w = w.t() if case["transpose"] else w
    pre = x @ w
    if case["bias"]:
        pre = pre + s["bias"].float()
    y = _act_plain(pre, case["epilogue"])
    if case["residual"]:
        y = y + s["residual"].float()
    out = dict(y=y.to(kind))
    if case["train"]:
        d = s["dy"].float()
        if case["epilogue"] != "none":
            d = d * _slope_plain(pre, case["epilogue"])
        out["dx"] = (d @ w.t()).to(kind)
        out["dw"] = (d.t() @ x if case["transpose"] else x.t() @ d).to(kind)
        if case["bias"]:
            out["db"] = d.sum(0).to(kind)
    return out


def _logp_plain(s):
    case, inv = s["case"], 1.0 / s["case"]["temperature"]
    x = s["logits"].float() * inv
    rows, c = x.shape
    at = s["labels"].long()
    given = at >= 0
    z = x - x.max(1, keepdim=True)[0]
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    mine = torch.gather(z, 1, at.clamp_min(0)[:, None]) - log_total
    out = dict(value=torch.where(given, mine[:, 0], torch.zeros_like(mine[:, 0])))
    live = e > 0
    if case["entropy"]:
        inside = torch.where(live, e * z, torch.zeros_like(e)).sum(1, keepdim=True)
        entropy = log_total - inside / total
        out["entropy"] = entropy[:, 0]
    if case["top"]:
        ids = torch.sort(s["logits"], dim=1, descending=True, stable=True)[1][:, :case["top"]]
        out["top_ids"] = ids.to(torch.int32)
        out["top_values"] = torch.gather(z, 1, ids) - log_total
    if case["train"]:
        p = e / total
        g = torch.where(given, s["dvalue"], torch.zeros_like(s["dvalue"]))[:, None] * inv
        d = -g * p
        d.scatter_add_(1, at.clamp_min(0)[:, None], g)
        if case["entropy"]:
            slope = torch.where(live, p * (z - log_total + entropy), torch.zeros_like(p))
            d = d - s["dentropy"][:, None] * inv * slope
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _distill_plain(s):
    case, inv = s["case"], 1.0 / s["case"]["temperature"]
    x = s["logits"].float() * inv
    z = x - x.max(1, keepdim=True)[0]
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    ids = s["ids"].long()
    live = ids >= 0
    t = torch.where(live, s["teacher"].float() * inv, torch.full_like(e[:, :1], -math.inf))
    t = t - t.max(1, keepdim=True)[0]
    q = torch.exp(t)
    weight = q.sum(1, keepdim=True)
    q = q / weight
    at = ids.clamp_min(0)
    gap = t - torch.log(weight) - (torch.gather(z, 1, at) - torch.log(total))
    out = dict(loss=torch.where(q > 0, q * gap, torch.zeros_like(q)).sum(1))
    if case["train"]:
        g = s["dloss"][:, None] * inv
        d = e / total * g
        d.scatter_add_(1, at, -q * g)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def run(state):
    if own:
        return _own_run(state)
    return dict(linear=_linear_plain, logp=_logp_plain,
                distill=_distill_plain)[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# The work of a pass, and its outputs from the definitions in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op, z, rows = case["op"], SIZE[case["dtype"]], case["rows"]
    if op == "linear":
        k, n = case["k"], case["n"]
        b = rows * k + k * n + rows * n * (2 if case["residual"] else 1) + n * case["bias"]
        f = 2 * rows * k * n
        if case["train"]:     # dy read; dx, dw and db written
            b += rows * n + rows * k + k * n + n * case["bias"]
            f *= 3
        return dict(bytes=z * b, flops=f)
    c = case["classes"]
    if op == "logp":
        b = z * rows * c + 8 * rows * (1 + case["top"]) + 4 * rows * case["entropy"]
        f = (4 + 2 * case["entropy"]) * rows * c
        if case["train"]:
            b, f = b + z * rows * c + 4 * rows * (1 + case["entropy"]), f + 4 * rows * c
        return dict(bytes=b, flops=f)
    k = case["k"]
    b, f = rows * (z * c + (z + 4) * k + 4), 4 * rows * c + 8 * rows * k
    if case["train"]:
        b, f = b + rows * (z * c + 4), f + 3 * rows * c
    return dict(bytes=b, flops=f)


def _act_exact(v, epilogue):
    """(activation, its derivative)."""
    one = torch.ones_like(v)
    if epilogue == "relu":
        return v.clamp_min(0.0), torch.where(v > 0, one, 0.0)
    if epilogue == "elu":
        return torch.where(v < 0, torch.expm1(v), v), torch.where(v < 0, torch.exp(v), one)
    if epilogue == "silu":
        p = torch.sigmoid(v)
        return v * p, p * (1 + v * torch.sigmoid(-v))
    if epilogue == "gelu":
        r = math.sqrt(2 / math.pi)
        t = torch.tanh(r * (v + GELU_CUBE * v ** 3))
        return (0.5 * v * (1 + t),
                0.5 * (1 + t) + 0.5 * v * (1 - t * t) * r * (1 + 3 * GELU_CUBE * v ** 2))
    return v, one


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = s["x"].double(), s["w"].double()
        if case["transpose"]:
            w = w.t().contiguous()
        pre = torch.mm(x, w)
        if case["bias"]:
            pre += s["bias"].double()
        y, slope = _act_exact(pre, case["epilogue"])
        if case["residual"]:
            y = y + s["residual"].double()
        out = dict(y=y)
        if case["train"]:
            d = slope * s["dy"].double()
            out["dx"] = torch.mm(d, w.t().contiguous())
            dw = torch.mm(x.t().contiguous(), d)
            out["dw"] = dw.t().contiguous() if case["transpose"] else dw
            if case["bias"]:
                out["db"] = d.sum(0)
        return out
    x = s["logits"].double() / case["temperature"]
    rows, c = x.shape
    if rows * c > 3 * 10 ** 8:
        return None
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(logp)
    row = torch.arange(rows, device=DEV)
    if case["op"] == "logp":
        at = s["labels"].long()
        given = at >= 0
        out = dict(value=torch.where(given, logp[row, at.clamp_min(0)], 0.0))
        if case["entropy"]:
            out["entropy"] = -torch.special.xlogy(p, p).sum(1)
        if case["top"]:
            rank = s["logits"].double()
            cols = torch.arange(c, device=DEV)
            picks = []
            for _ in range(case["top"]):   # the largest left, the lowest index among equals
                best = rank.max(1, keepdim=True)[0]
                picks.append(torch.where(rank == best, cols, c).min(1)[0])
                rank[row, picks[-1]] = -math.inf
            ids = torch.stack(picks, 1)
            out["top_ids"] = ids.int()
            out["top_values"] = logp[row[:, None], ids]
        if case["train"]:
            g = torch.where(given, s["dvalue"].double(), 0.0) / case["temperature"]
            d = -p * g[:, None]
            d[row, at.clamp_min(0)] += g
            if case["entropy"]:
                h = s["dentropy"].double() / case["temperature"]
                d -= h[:, None] * (torch.special.xlogy(p, p) + p * out["entropy"][:, None])
            out["dlogits"] = d
        return out
    ids = s["ids"].long()
    t = torch.where(ids >= 0, s["teacher"].double() / case["temperature"], -math.inf)
    q = torch.softmax(t, 1)
    at = ids.clamp_min(0)
    chosen = logp[row[:, None], at]
    out = dict(loss=(torch.special.xlogy(q, q) - torch.where(q > 0, q * chosen, 0.0)).sum(1))
    if case["train"]:
        g = s["dloss"].double()[:, None] / case["temperature"]
        d = p * g
        for j in range(case["k"]):
            d[row, at[:, j]] -= (q * g)[:, j]
        out["dlogits"] = d
    return out
