"""Layer norm, forward and backward, on the GPU against 64 bits.

Tolerances (u = 2^-24): a row's sum of c values is added in chains of at most
16 per thread (more in rows over 16,384: c / 8,192) and a tree, so the mean is
off by D u avg|x|, D = 32 + c / 4096; the deviations by that and u |d|; the
variance by 2 of those and D u relative, rstd by half of it; each later
operation by u.  Columns' sums over rows: chains of at most rows / 1024 + 64.
The result is then rounded to its type: half a step."""
import pytest
import torch

from expert_cases import DTYPES, U, gen, half_step, least, padded, randn, within

pytestmark = pytest.mark.gpu


def reference(x, gamma, beta, eps, dy=None):
    x64 = x.double()
    c = x.shape[1]
    g = torch.ones(c, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    mean = x64.mean(1, keepdim=True)
    d = x64 - mean
    var = (d * d).mean(1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    xh = d * r
    deep = 32 + c / 4096
    dm = deep * U * x64.abs().mean(1, keepdim=True) + U * mean.abs()
    # rstd: relative, from the deviations' shift (2 dm |d| averaged, over var + eps)
    dr = deep * U + dm * d.abs().mean(1, keepdim=True) * r * r + dm * dm * r * r + 4 * U
    dxh = dm * r + xh.abs() * (dr + 4 * U)
    out = dict(y=xh * g + b, y_tol=dxh * g.abs() + 3 * U * ((xh * g).abs() + b.abs()),
               mean=mean[:, 0], mean_tol=dm[:, 0], rstd=r[:, 0], rstd_tol=(r * dr)[:, 0])
    if dy is not None:
        t = dy.double() * g
        m0, m1 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
        a0, a1 = t.abs().mean(1, keepdim=True), (t * xh).abs().mean(1, keepdim=True)
        out["dx"] = r * (t - m0 - xh * m1)
        terms = t.abs() + a0 + xh.abs() * a1
        out["dx_tol"] = (r * (deep * U * terms + dxh * a1
                              + xh.abs() * (t.abs() * dxh).mean(1, keepdim=True))
                         + (dr + 4 * U) * r * terms)
        long = (96 + x.shape[0] / 256) * U
        out["dgamma"] = (dy.double() * xh).sum(0)
        out["dgamma_tol"] = (long * (dy.double() * xh).abs().sum(0)
                             + (dy.double().abs() * dxh).sum(0))
        out["dbeta"] = dy.double().sum(0)
        out["dbeta_tol"] = long * dy.double().abs().sum(0)
    return out


def check(got, ref, name, dtype):
    want = ref[name]
    within(got, want, ref[name + "_tol"] + half_step(dtype) * (want.abs() + ref[name + "_tol"])
           + least(dtype), name)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 256), (7, 63), (5, 64), (130, 65),
                                       (9, 255), (33, 1023), (6, 1024), (5, 1025), (3, 4096),
                                       (4, 4097), (2, 16384), (3, 16385), (2, 70001),
                                       (5000, 41), (2708, 1433), (9001, 200)])
def test_norm(gpu, dtype, rows, cols):
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(rows * 31 + cols)
    x = padded(randn(g, (rows, cols), dt, 2.0) + 3.0, 3)
    dy = padded(randn(g, (rows, cols), dt), 5)
    gamma, beta = 1 + randn(g, cols, dt, 0.3), randn(g, cols, dt)
    ref = reference(x, gamma, beta, 1e-5, dy)
    y, mean, rstd = tg.layer_norm(x, gamma, beta, 1e-5, with_stats=True)
    check(y, ref, "y", dt)
    check(mean, ref, "mean", torch.float32)
    check(rstd, ref, "rstd", torch.float32)
    dx, dgamma, dbeta = tg.layer_norm_backward(dy, x, mean, rstd, gamma)
    for name, v in dict(dx=dx, dgamma=dgamma, dbeta=dbeta).items():
        check(v, ref, name, dt)
    again = tg.layer_norm_backward(dy, x, mean, rstd, gamma)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dgamma, dbeta)))


@pytest.mark.parametrize("gamma,beta", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_norm_weights(gpu, dtype, gamma, beta):
    """Weights that are missing, and float32 weights of 16-bit rows."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(5)
    x, dy = randn(g, (37, 300), dt), randn(g, (37, 300), dt)
    w = randn(g, 300, torch.float32) if gamma else None
    b = randn(g, 300, torch.float32) if beta else None
    ref = reference(x, w, b, 1e-3, dy)
    y, mean, rstd = tg.layer_norm(x, w, b, 1e-3, with_stats=True)
    check(y, ref, "y", dt)
    dx, dgamma, dbeta = tg.layer_norm_backward(dy, x, mean, rstd, w)
    kind = torch.float32 if gamma else dt
    assert dgamma.dtype == kind and dbeta.dtype == kind
    check(dx, ref, "dx", dt)
    check(dgamma, ref, "dgamma", kind)
    check(dbeta, ref, "dbeta", kind)


def test_norm_in_place_and_no_rows(gpu):
    import tinygnn_amd as tg
    g = gen(6)
    for cols in (40, 3000, 20000):
        x, dy = randn(g, (50, cols), torch.float32), randn(g, (50, cols), torch.float32)
        y, mean, rstd = tg.layer_norm(x, with_stats=True)
        want = tg.layer_norm_backward(dy, x, mean, rstd)
        x2, dy2 = x.clone(), dy.clone()
        assert tg.layer_norm_backward(dy2, x, mean, rstd, out=dy2)[0] is dy2
        assert torch.equal(dy2, want[0])
        assert tg.layer_norm(x2, out=x2) is x2 and torch.equal(x2, y)
    x = torch.empty(0, 33, device="cuda")
    y, mean, rstd = tg.layer_norm(x, with_stats=True)
    dx, dgamma, dbeta = tg.layer_norm_backward(x, x, mean, rstd)
    assert y.shape == dx.shape == (0, 33)
    assert not dgamma.any() and not dbeta.any()


def test_norm_constant_and_bad_rows(gpu):
    """A constant row is beta; NaN and infinities stay in their rows."""
    import tinygnn_amd as tg
    x = torch.full((4, 500), 1e4, device="cuda")
    x[1] = torch.randn(500, device="cuda", generator=gen(1))
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    beta = torch.randn(500, device="cuda", generator=gen(2))
    y = tg.layer_norm(x, None, beta)
    assert torch.equal(y[0], beta)
    assert torch.isfinite(y[1]).all() and torch.isnan(y[2]).all() and torch.isnan(y[3, 4])


def test_norm_gradient_by_differences(gpu):
    """The backward pass against central differences of the forward formula in
    64 bits: third derivatives of order 10 and steps of 1e-4 leave 1e-7."""
    import tinygnn_amd as tg
    g = gen(7)
    x, dy = randn(g, (3, 17), torch.float32), randn(g, (3, 17), torch.float32)
    gamma = randn(g, 17, torch.float32)
    _, mean, rstd = tg.layer_norm(x, gamma, with_stats=True)
    dx, dgamma, _ = tg.layer_norm_backward(dy, x, mean, rstd, gamma)

    def loss(xv, gv):
        return (reference(xv, gv, None, 1e-5)["y"] * dy.double()).sum()

    for at, grad, of in ((x, dx, 0), (gamma, dgamma, 1)):
        for i in range(0, at.numel(), 5):
            step = torch.zeros(at.numel(), dtype=torch.float64, device="cuda")
            step[i] = 1e-4
            v = [x.double(), gamma.double()]
            lo, hi = list(v), list(v)
            hi[of] = v[of] + step.view(at.shape)
            lo[of] = v[of] - step.view(at.shape)
            want = (loss(*hi) - loss(*lo)) / 2e-4
            assert abs(grad.flatten()[i].item() - want.item()) < 2e-5 * (1 + abs(want.item()))


def test_norm_of_more_rows_than_a_launch_takes(gpu):
    """2^22 rows and some, of 1,024 threads each: 2^32 threads and more."""
    import tinygnn_amd as tg
    rows, cols = 2 ** 22 + 300, 2052
    x = torch.empty(rows, cols, device="cuda")
    some = torch.tensor([0, 1, 2 ** 22 - 2, 2 ** 22 - 1, 2 ** 22, rows - 1], device="cuda")
    values = randn(gen(4), (len(some), cols), torch.float32)
    x[some] = values
    y, mean, rstd = tg.layer_norm(x, with_stats=True, out=x)
    want, want_mean, want_rstd = tg.layer_norm(values, with_stats=True)
    assert torch.equal(y[some], want)
    assert torch.equal(mean[some], want_mean) and torch.equal(rstd[some], want_rstd)
