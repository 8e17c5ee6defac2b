"""Plain 64-bit forms of the dense layers, the log probabilities and the
distillation, with bounds of what float32 operations may be off by."""
import math

import torch

from expert_cases import U, half_step, least

INF = float("inf")


def in_range(got, want, tol):
    """got, an infinity taken for `want` where a value that the bound allows lies
    past the largest float32: the logits' lowest value under the largest makes
    terms of twice that size, and |want| + tol >= 2^128 (1 - 2^-25) rounds to infinity."""
    reach = want.double().abs() + tol >= 2.0 ** 128 * (1 - 2.0 ** -25)
    same = torch.isinf(got) & torch.isfinite(want) & (got.sign() == want.sign())
    return torch.where(reach & same, want, got.double())


# ---------------------------------------------------------------------------
# Dense layers
# ---------------------------------------------------------------------------
def _inner(v, name):
    """(s, ds/dv) of the activations v sigmoid(s)."""
    if name == "silu":
        return v, torch.ones_like(v)
    c = 2 * math.sqrt(2 / math.pi)
    return c * (v + 0.044715 * v ** 3), c * (1 + 3 * 0.044715 * v ** 2)


def act(v, name):
    """(activation, its derivative, bounds of both from evaluating them in float32).

    sigmoid(s): s of a few operations is off by 6 u |s|, exp of it by that and
    2 u, the sum and the reciprocal by 3 u: relative (6 |s| + 6) u at most."""
    one = torch.ones_like(v)
    if name == "none":
        return v, one, 0 * v, 0 * v
    if name == "relu":
        return v.clamp_min(0), (v > 0).double(), 0 * v, 0 * v
    if name == "elu":
        y = torch.where(v < 0, torch.expm1(v), v)
        e = torch.where(v < 0, torch.exp(v), one)
        # (expm1's difference: an exp off by 2^-23 of its own, of a value over 0.29)
        return y, e, 16 * U * y.abs(), torch.where(v < 0, (2 * v.abs() + 4) * U * e, 0.0)
    s, ds = _inner(v, name)
    p, r = torch.sigmoid(s), torch.sigmoid(-s)
    rel = (6 * s.abs() + 6) * U
    y = v * p
    slope = p + v * p * r * ds
    # 1 - p is off by p's own error and u, absolutely
    bad = rel * p + (v * ds).abs() * p * (rel * (r + p) + U + 4 * U * r) + 2 * U * slope.abs()
    return y, slope, (rel + 2 * U) * y.abs(), bad


def linear(x, w, bias, name, residual, transpose):
    """y, pre and their bounds before the last rounding."""
    w = w.double().t().contiguous() if transpose else w.double()
    x = x.double()
    pre, size = x @ w, x.abs() @ w.abs()
    if bias is not None:
        pre, size = pre + bias.double(), size + bias.double().abs()
    off = (x.shape[1] + 2) * U * size
    y, slope, bad, _ = act(pre, name)
    # slopes are below 1.13, and within `off` of a corner the values are
    tol = 1.13 * off + bad
    if residual is not None:
        y = y + residual.double()
        tol = tol + 2 * U * y.abs()
    return y, tol, pre, off


def linear_backward(dy, x, w, pre, name, transpose, dtype):
    """{dx, dw, db: (value, bound)} from the given pre."""
    x, dy = x.double(), dy.double()
    w = w.double().t().contiguous() if transpose else w.double()
    d, bad = dy, 0 * dy
    if name != "none":
        _, slope, _, off = act(pre.double(), name)
        d = dy * slope
        bad = dy.abs() * off + U * d.abs()
    rounded = bad if name == "none" else bad + half_step(dtype) * (d.abs() + bad) + least(dtype)
    m, n = d.shape
    wt, xt = w.t().contiguous(), x.t().contiguous()
    dx = d @ wt, rounded @ wt.abs() + (n + 2) * U * (d.abs() @ wt.abs())
    dw = xt @ d, xt.abs() @ rounded + (m + 2) * U * (xt.abs() @ d.abs())
    if transpose:
        dw = dw[0].t(), dw[1].t()
    db = d.sum(0), bad.sum(0) + (m + 2) * U * d.abs().sum(0)
    return dict(dx=dx, dw=dw, db=db)


def rounded(value, tol, dtype):
    """The bound with the result's own rounding."""
    return tol + half_step(dtype) * (value.abs() + tol) + least(dtype)


# ---------------------------------------------------------------------------
# Log probabilities, distillation
# ---------------------------------------------------------------------------
class Row:
    """log p of every class, and bounds: `sum` of log s, `at` of log p.

    z = (x - m) / T is off by 4 u |z|, exp of it by that, 2 u |z| and 2 u more;
    a sum of positive terms (chains of 256 at most and a tree) by 300 u: s by
    (6 E|z| + 304) u relative, log s by that and 2 u of itself."""

    def __init__(self, logits, temperature):
        x = logits.double()
        self.nan = (torch.isnan(x) | (x == INF)).any(1)
        self.m = torch.where(torch.isnan(x), -INF, x).max(1, keepdim=True)[0]
        self.empty = (self.m[:, 0] == -INF) & ~self.nan
        z = torch.where(x == -INF, -INF, (x - self.m) / temperature)
        z[self.empty | self.nan] = 0.0
        e = torch.exp(z)
        s = e.sum(1, keepdim=True)
        self.p = e / s
        self.log_s = torch.log(s)
        self.logp = z - self.log_s
        fine = torch.where(z > -INF, z.abs(), 0.0)
        self.mean_z = (self.p * fine).sum(1, keepdim=True)
        self.sum = (6 * self.mean_z + 304) * U + 2 * U * self.log_s
        self.at = self.sum + 4 * U * fine + U * torch.where(z > -INF, self.logp.abs(), 0.0)
        self.entropy = -(torch.special.xlogy(self.p, self.p)).sum(1)
        # the sum of p z: each term off by exp's and z's, the whole by s's
        self.entropy_tol = ((self.sum + 304 * U) * (1 + self.mean_z))[:, 0] \
            + 12 * U * (self.p * fine * (fine + 1)).sum(1) + 4 * U * self.entropy


def labels_of(labels, row, n):
    """(at, given): the label's column and whether there is one."""
    given = (labels >= 0) & (labels < n)
    return torch.where(given, labels, 0).long(), given


def value(row, labels):
    at, given = labels_of(labels, row, row.p.shape[1])
    v = torch.gather(row.logp, 1, at[:, None])[:, 0]
    v = torch.where(row.empty, -INF, v)
    v = torch.where(row.nan, float("nan"), v)
    tol = torch.gather(row.at, 1, at[:, None])[:, 0]
    return torch.where(given, v, 0.0), tol


def top(logits, k):
    """Columns of the k largest, the lower first among equals; -1: none."""
    x = torch.where(torch.isnan(logits.double()), -INF, logits.double()).clone()
    cols = torch.arange(x.shape[1], device=x.device)
    rows = torch.arange(x.shape[0], device=x.device)
    out = []
    for _ in range(k):
        best = x.max(1, keepdim=True)[0]
        first = torch.where(x == best, cols, x.shape[1]).min(1)[0]
        out.append(torch.where(best[:, 0] > -INF, first, -1))
        x[rows, first] = -INF
    return torch.stack(out, 1)


def backward(row, labels, dvalue, dentropy, temperature):
    """(dlogits, bound) before rounding."""
    p = row.p
    d, tol = torch.zeros_like(p), torch.zeros_like(p)
    zero = torch.ones_like(row.nan)
    rel = row.at + 6 * U
    if dvalue is not None:
        at, given = labels_of(labels, row, p.shape[1])
        g = torch.where(given, dvalue.double(), 0.0) / temperature
        zero &= g == 0
        hit = torch.zeros_like(p)
        hit[torch.arange(len(at), device=p.device), at] = g
        d += hit - g[:, None] * p
        tol += g.abs()[:, None] * p * rel + 4 * U * (hit.abs() + g.abs()[:, None] * p)
    if dentropy is not None:
        h = dentropy.double()[:, None] / temperature
        zero &= h[:, 0] == 0
        inner = torch.where(p > 0, row.logp, 0.0) + row.entropy[:, None]
        size = torch.where(p > 0, row.logp.abs(), 0.0) + row.entropy[:, None]
        d -= h * p * inner
        tol += h.abs() * p * (rel * size + row.at + row.entropy_tol[:, None] + 6 * U * size)
    d[row.nan] = float("nan")
    d[zero | row.empty] = 0.0
    return d, tol


def distill(row, teacher, ids, temperature, dloss=None):
    """(loss, its bound), and with dloss (dlogits, its bound)."""
    n = row.p.shape[1]
    live = (ids >= 0) & (ids < n)
    t = torch.where(live, teacher.double(), -INF)
    none = ~(t > -INF).any(1) & ~torch.isnan(t).any(1)
    tm = torch.where(torch.isnan(t), -INF, t).max(1, keepdim=True)[0]
    z = torch.where(t == -INF, -INF, (t - tm) / temperature)
    z[none] = 0.0
    e = torch.exp(z)
    q = torch.where(none[:, None], 0.0, e / e.sum(1, keepdim=True))
    log_q = z - torch.log(e.sum(1, keepdim=True))
    fine = torch.where(z > -INF, z.abs(), 0.0)
    rel = (6 * fine + 6 * (q * fine).sum(1, keepdim=True) + ids.shape[1] + 16) * U
    at = torch.where(live, ids, 0).long()
    logp = torch.gather(row.logp, 1, at)
    logp = torch.where(row.empty[:, None], -INF, logp)
    gap = torch.where(q == 0, 0.0, q * (log_q - logp))
    loss = gap.sum(1)
    loss = torch.where(row.nan & ~none, float("nan"), loss)
    size = torch.where(q > 0, log_q.abs() + torch.where(logp > -INF, logp.abs(), 0.0), 0.0)
    tol = (q * (rel * (1 + size) + torch.gather(row.at, 1, at) + 4 * U * size)).sum(1) \
        + ids.shape[1] * U * (q * size).sum(1)
    if dloss is None:
        return loss, tol
    g = dloss.double()[:, None] / temperature
    d = g * row.p
    dt = g.abs() * row.p * (row.at + 6 * U)
    for j in range(ids.shape[1]):
        add = torch.zeros_like(d).scatter_(1, at[:, j:j + 1], (g * q)[:, j:j + 1])
        d = d - add
        dt = dt + add.abs() * (rel[:, j:j + 1] + (ids.shape[1] + 4) * U)
    dt = dt + 4 * U * g.abs() * row.p
    d[(row.nan | torch.isnan(q).any(1))] = float("nan")
    d[none | row.empty | (dloss == 0)] = 0.0
    return loss, tol, d, dt
